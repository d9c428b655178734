"""Cases of the digital operators that stand around the analog tiles of a transformer block: layer norm (with the residual
sum and the dropout in front of it), dropout from a counter-based generator, and low-rank adapters of many requests beside a
shared projection.

``run`` computes them in elementary torch operations, or - where ``own`` is true - through ``aihwkit_b200.digital``.
``exact`` gives the same results from the definitions in 64 bits.  Sizes are those of the GPT-2-shaped inference (768,
2304), of the mapped benchmark layer (4096) and of the single-tile ones (1024, 785), and odd ones beside them.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5
MOST_VALUES = 8192 * 4096  # of one activation of a case that trains; twice that where nothing does


# ---- the cases ---------------------------------------------------------------------------------------------------------


def _norm(name, rows, cols, dtype, train, residual, p=0.0):
    return {"name": name, "op": "norm", "rows": rows, "cols": cols, "dtype": dtype, "train": train, "residual": residual, "p": p}


def _dropout(name, rows, cols, dtype, train, residual, p):
    return {"name": name, "op": "dropout", "rows": rows, "cols": cols, "dtype": dtype, "train": train, "residual": residual, "p": p}


def _adapters(name, rows, requests, adapters, k, n, rank, dtype, train, ragged):
    return {"name": name, "op": "adapters", "rows": rows, "requests": requests, "adapters": adapters, "k": k, "n": n,
            "rank": rank, "dtype": dtype, "train": train, "ragged": ragged}


def listed():
    return [
        # one token of one sequence: the sum with the residual stream and the norm in front of the next layer
        _norm("norm_one_token", 1, 768, "f32", False, True),
        # the same for a batch of prompts, 16 x 1024 tokens
        _norm("norm_prompts", 16384, 768, "f32", False, True),
        # a training step of a wide block, dropout in front of the residual sum, forward and backward
        _norm("norm_train_wide", 8192, 4096, "bf16", True, True, 0.1),
        # rows that no vector load divides
        _norm("norm_train_odd", 5003, 785, "f16", True, False),
        # a short batch in front of one layer
        _dropout("dropout_small", 64, 768, "f32", False, False, 0.1),
        # the branch of a block, added to its residual stream, forward and backward
        _dropout("dropout_train_residual", 16384, 768, "f32", True, True, 0.1),
        # the widest activation of a step
        _dropout("dropout_wide", 16384, 4096, "bf16", False, False, 0.25),
        # one token of one request
        _adapters("adapters_one_token", 1, 1, 4, 768, 2304, 8, "f32", False, False),
        # a decoding step of many requests, each with one of many adapters
        _adapters("adapters_decode", 256, 256, 64, 4096, 4096, 16, "bf16", False, False),
        # prompts of many lengths, some without an adapter
        _adapters("adapters_prompts", 16384, 16, 8, 768, 2304, 16, "f32", False, True),
        # adapters in training beside a wide projection
        _adapters("adapters_train", 8192, 8, 2, 4096, 4096, 32, "bf16", True, True),
        # odd widths, odd rank
        _adapters("adapters_train_odd", 4099, 5, 3, 785, 461, 5, "f16", True, True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "dropout", "adapters", "adapters"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    train = rng.random() < 0.5
    most = MOST_VALUES if train or op == "norm" else 2 * MOST_VALUES
    if dtype == "f32":
        most //= 2
    while True:
        rows = _spread(rng, 1, 16384)
        if op != "adapters":
            cols = _spread(rng, 33, 4096)
            if rng.random() < 0.6:
                cols = max(64, cols // 64 * 64)
            if rows * cols > most:
                continue
            case = {"op": op, "rows": rows, "cols": cols, "dtype": dtype, "train": train, "residual": rng.random() < 0.5}
            if op == "norm":
                case["p"] = rng.choice([0.0, 0.1, 0.3]) if case["residual"] and train else 0.0
            else:
                case["p"] = rng.choice([0.05, 0.1, 0.25, 0.5])
            return case
        k, n = _spread(rng, 65, 4096), _spread(rng, 65, 4096)
        if rng.random() < 0.6:
            k, n = max(64, k // 64 * 64), max(64, n // 64 * 64)
        if rows * max(k, n) > most:
            continue
        ragged = train or (rows > 16 and rng.random() < 0.7)
        if not ragged:
            rows = min(rows, 256)
        rank = rng.choice([1, 4, 5, 8, 16, 16, 32, 64]) if dtype != "f32" else rng.choice([1, 4, 5, 8, 16, 16, 24])
        return {"op": op, "rows": rows, "requests": _spread(rng, 1, min(8, rows)) if ragged else rows,
                "adapters": _spread(rng, 1, 16), "k": k, "n": n, "rank": rank, "dtype": dtype, "train": train, "ragged": ragged}


# ---- what a user's program has in hand ---------------------------------------------------------------------------------


def _generator(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(int(seed))


def _normal(gen, shape, dtype, std=1.0, mean=0.0):
    t = torch.empty(shape, dtype=torch.float32, device="cuda").normal_(mean, std, generator=gen)
    return t.to(DTYPES[dtype])


def _inputs(case, seed):
    gen = _generator(seed)
    dtype = case["dtype"]
    if case["op"] != "adapters":
        rows, cols = case["rows"], case["cols"]
        s = {"x": _normal(gen, (rows, cols), dtype)}
        if case["residual"]:
            # a residual stream: an offset, and a few channels far larger than the others
            loud = 1.0 + 9.0 * (torch.rand(cols, device="cuda", generator=gen) < 0.01)
            s["residual"] = (torch.empty(rows, cols, device="cuda").normal_(0.2, 1.5, generator=gen) * loud).to(DTYPES[dtype])
        if case["op"] == "norm":
            s["weight"] = torch.empty(cols, device="cuda").normal_(1.0, 0.2, generator=gen)
            s["bias"] = torch.empty(cols, device="cuda").normal_(0.0, 0.1, generator=gen)
        if case["train"]:
            s["gy"] = _normal(gen, (rows, cols), dtype)
            if case["op"] == "norm" and case["residual"]:
                s["gh"] = _normal(gen, (rows, cols), dtype)
        s["seed"], s["call"] = 1000003 * int(seed) + 12345678901, int(seed) % 1000
        return s
    rows, k, n, rank, requests = case["rows"], case["k"], case["n"], case["rank"], case["requests"]
    host = np.random.default_rng([int(seed), 7])
    if case["ragged"]:
        # lengths of all sizes, rows behind the last request that belong to none
        weights = np.exp(host.uniform(0.0, 3.0, requests))
        used = rows - rows // 50
        starts = np.concatenate([[0], np.cumsum(np.floor(weights / weights.sum() * used).astype(np.int64))])
    else:
        starts = np.arange(requests + 1)
    ids = host.integers(0, case["adapters"], requests)
    if requests > 2:
        ids[host.random(requests) < 0.1] = -1
    return {"x": _normal(gen, (rows, k), dtype), "base": _normal(gen, (rows, n), dtype),
            "a": _normal(gen, (case["adapters"], rank, k), dtype, 1.0 / math.sqrt(k)),
            "b": _normal(gen, (case["adapters"], rank, n), dtype, 1.0 / math.sqrt(rank)),
            "scale": torch.empty(case["adapters"], device="cuda").uniform_(0.5, 2.0, generator=gen),
            "host_starts": [int(v) for v in starts], "host_ids": [int(v) for v in ids],
            "starts": torch.tensor(starts, dtype=torch.int32, device="cuda"),
            "ids": torch.tensor(ids, dtype=torch.int32, device="cuda"),
            **({"gy": _normal(gen, (rows, n), dtype)} if case["train"] else {})}


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = dict(case)
    if case["train"]:  # what a step differentiates
        names = ("x", "a", "b") if case["op"] == "adapters" else ("x", "residual", "weight", "bias")
        state["leaves"] = {k: state[k].requires_grad_(own) for k in names if k in state}
    return state


# ---- plain forms -------------------------------------------------------------------------------------------------------

TAG_HIGH, TAG_LOW = 0xB0000000, 0xB0000001


def _philox(block, call, tag, seed):
    """Philox4x32 with ten rounds on 64-bit integers: four 32-bit words per block."""
    mask = 0xFFFFFFFF
    c0, c1 = block & mask, block >> 32
    c2, c3 = torch.full_like(block, call & mask), torch.full_like(block, tag)
    k0, k1 = seed & mask, (seed >> 32) & mask

    def product(m, c):  # high and low word of a 32 x 32 bit product, in pieces that 64 bits hold
        return (m * (c >> 16) + ((m * (c & 0xFFFF)) >> 16)) >> 16, (m * c) & mask

    for _ in range(10):
        h0, l0 = product(0xD2511F53, c0)
        h1, l1 = product(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    return torch.stack([c0, c1, c2, c3], dim=-1)


def _kept(rows, cols, p, seed, call):
    """Which elements of [rows, cols] a dropout of probability p leaves."""
    per_row = (cols + 7) // 8
    block = torch.arange(rows * per_row, dtype=torch.int64, device="cuda")
    high, low = _philox(block, call, TAG_HIGH, seed), _philox(block, call, TAG_LOW, seed)
    lanes = torch.stack([(high & 0xFFFF) << 16 | (low & 0xFFFF), (high >> 16) << 16 | low >> 16], dim=-1)
    return lanes.reshape(rows, per_row * 8)[:, :cols] >= int(round(p * 2.0 ** 32))


def _drop(x, kept, p):
    return torch.where(kept, x * (1.0 / (1.0 - p)), torch.zeros_like(x))


def _plain_norm(s, case):
    dtype, p = DTYPES[case["dtype"]], case["p"]
    h = s["x"].float()
    kept = _kept(case["rows"], case["cols"], p, s["seed"], s["call"]) if p > 0 else None
    if kept is not None:
        h = _drop(h, kept, p)
    if case["residual"]:
        h = h + s["residual"].float()
    centred = h - h.mean(dim=-1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(dim=-1, keepdim=True) + EPS)
    unit = centred * rstd
    out = {"y": (unit * s["weight"] + s["bias"]).to(dtype)}
    if case["residual"]:
        out["h"] = h.to(dtype)
    if case["train"]:
        gy = s["gy"].float()
        t = gy * s["weight"]
        dh = rstd * (t - t.mean(dim=-1, keepdim=True) - unit * (t * unit).mean(dim=-1, keepdim=True))
        if case["residual"]:
            dh = dh + s["gh"].float()
            out["dresidual"] = dh.to(dtype)
        out["dx"] = (dh if kept is None else _drop(dh, kept, p)).to(dtype)
        out["dweight"], out["dbias"] = (gy * unit).sum(dim=0), gy.sum(dim=0)
    return out


def _plain_dropout(s, case):
    dtype, p = DTYPES[case["dtype"]], case["p"]
    kept = _kept(case["rows"], case["cols"], p, s["seed"], s["call"])
    y = _drop(s["x"].float(), kept, p)
    out = {"y": (y + s["residual"].float() if case["residual"] else y).to(dtype)}
    if case["train"]:
        out["dx"] = _drop(s["gy"].float(), kept, p).to(dtype)
    return out


def _plain_adapters(s, case):
    dtype = DTYPES[case["dtype"]]
    x, a, b, scale = s["x"].float(), s["a"].float(), s["b"].float(), s["scale"]
    y = s["base"].float()
    gy = s["gy"].float() if case["train"] else None
    dx, da, db = (torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)) if case["train"] else (None, None, None)
    if not case["ragged"] and not case["train"]:  # one row each: gathered adapters, one batched product each
        ids = s["ids"].long()
        known = ids.clamp(min=0)
        v = (a[known] * x.unsqueeze(1)).sum(dim=2)
        delta = (v.unsqueeze(2) * b[known]).sum(dim=1) * scale[known].unsqueeze(1)
        return {"y": torch.where((ids >= 0).unsqueeze(1), y + delta, y).to(dtype)}
    y = y.clone()
    for j, i in enumerate(s["host_ids"]):
        begin, end = s["host_starts"][j], s["host_starts"][j + 1]
        if i < 0 or begin == end:
            continue
        v = x[begin:end] @ a[i].t()
        y[begin:end] += scale[i] * (v @ b[i])
        if case["train"]:
            u = scale[i] * (gy[begin:end] @ b[i].t())
            dx[begin:end] = u @ a[i]
            da[i] += u.t() @ x[begin:end]
            db[i] += scale[i] * (v.t() @ gy[begin:end])
    out = {"y": y.to(dtype)}
    if case["train"]:
        out.update(dx=dx.to(dtype), da=da.to(dtype), db=db.to(dtype))
    return out


# ---- the framework's calls ---------------------------------------------------------------------------------------------


def _own(s, case):
    from aihwkit_b200 import digital

    if case["op"] == "norm":
        if case["residual"]:
            y, h = digital.add_layer_norm(s["x"], s["residual"], s["weight"], s["bias"], EPS, p=case["p"], seed=s["seed"],
                                          call=s["call"])
            out = {"y": y, "h": h}
        else:
            out = {"y": digital.layer_norm(s["x"], s["weight"], s["bias"], EPS)}
        if case["train"]:
            names = [k for k in ("x", "residual", "weight", "bias") if k in s]
            results, grads = [out["y"]], [s["gy"]]
            if case["residual"]:
                results.append(out["h"])
                grads.append(s["gh"])
            found = torch.autograd.grad(results, [s[k] for k in names], grads)
            out.update({"d" + k: g for k, g in zip(names, found)})
    elif case["op"] == "dropout":
        out = {"y": digital.dropout(s["x"], case["p"], seed=s["seed"], call=s["call"], residual=s.get("residual"))}
        if case["train"]:
            out["dx"], = torch.autograd.grad([out["y"]], [s["x"]], [s["gy"]])
    else:
        out = {"y": digital.low_rank_add(s["base"], s["x"], s["a"], s["b"], s["scale"], s["ids"], s["starts"])}
        if case["train"]:
            out["dx"], out["da"], out["db"] = torch.autograd.grad([out["y"]], [s["x"], s["a"], s["b"]], [s["gy"]])
    return {k: v.detach() for k, v in out.items()}


def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    return {"norm": _plain_norm, "dropout": _plain_dropout, "adapters": _plain_adapters}[case["op"]](state, case)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] != "adapters":
        values = case["rows"] * case["cols"]
        norm = case["op"] == "norm"
        moved = 2 + (1 if case["residual"] else 0) + (1 if norm and case["residual"] else 0)  # x, y, residual, h
        if case["train"]:
            moved += 2  # gy, dx
            if norm and case["residual"]:
                moved += 2 if case["p"] > 0 else 1  # gh, and the residual's gradient where dropout sets it apart
        flops = values * ((8 if norm else 2) + ((14 if norm else 2) if case["train"] else 0))
        return {"bytes": values * moved * size + (case["cols"] * 4 * (4 if case["train"] else 2) if norm else 0), "flops": flops}
    rows, k, n, rank = case["rows"], case["k"], case["n"], case["rank"]
    adapters = min(case["adapters"], case["requests"]) * rank * (k + n)
    moved = rows * (k + 2 * n) + adapters
    flops = 2.0 * rows * rank * (k + n)
    if case["train"]:
        moved += rows * (n + k) + case["adapters"] * rank * (k + n)  # gy, dx, the adapters' gradients
        flops *= 3
    return {"bytes": moved * size, "flops": flops}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------


def _exact_kept(rows, cols, p, seed, call):
    """The kept elements, drawn with numpy's 64-bit integers; the low half-words only where the high ones tie."""
    word = np.uint64(0xFFFFFFFF)
    threshold = round(p * 4294967296.0)
    per_row = -(-cols // 8)

    def words(blocks, tag):
        counter = [blocks & word, blocks >> np.uint64(32), np.full_like(blocks, call), np.full_like(blocks, tag)]
        key = [seed % 2 ** 32, seed // 2 ** 32 % 2 ** 32]
        for _ in range(10):
            first, second = counter[0] * np.uint64(0xD2511F53), counter[2] * np.uint64(0xCD9E8D57)
            counter = [second >> np.uint64(32) ^ counter[1] ^ np.uint64(key[0]), second & word,
                       first >> np.uint64(32) ^ counter[3] ^ np.uint64(key[1]), first & word]
            key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
        return np.stack(counter, axis=1).astype("<u4").view("<u2")  # eight half-words a block

    kept = np.empty((rows, cols), dtype=bool)
    step = max(1, (1 << 21) // per_row)
    for r in range(0, rows, step):
        e = min(rows, r + step)
        blocks = np.arange(r * per_row, e * per_row, dtype=np.uint64)
        high = words(blocks, TAG_HIGH).astype(np.int64)
        keep = high > threshold >> 16
        tied = (high == threshold >> 16).any(axis=1)
        if tied.any():
            full = (high[tied] << 16) + words(blocks[tied], TAG_LOW)
            keep[tied] = full >= threshold
        kept[r:e] = keep.reshape(e - r, per_row * 8)[:, :cols]
    return torch.from_numpy(kept).cuda()


def exact(case, seed):
    s = _inputs(case, seed)
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if case["op"] == "adapters":
        factor = torch.zeros(case["rows"], case["adapters"], dtype=torch.float64, device="cuda")  # rows' scales, per adapter
        for j, i in enumerate(s["host_ids"]):
            if i >= 0:
                factor[s["host_starts"][j]:s["host_starts"][j + 1], i] = d["scale"][i]
        y = d["base"]
        dx = torch.zeros_like(d["x"])
        da, db = torch.zeros_like(d["a"]), torch.zeros_like(d["b"])
        for i in range(case["adapters"]):
            rows = factor[:, i].nonzero().flatten()
            x, f = d["x"][rows], factor[rows, i:i + 1]
            v = torch.einsum("mk,rk->mr", x, d["a"][i]) * f
            y = y.index_add(0, rows, torch.einsum("mr,rn->mn", v, d["b"][i]))
            if case["train"]:
                gy = d["gy"][rows]
                u = torch.einsum("mn,rn->mr", gy, d["b"][i]) * f
                dx[rows] = torch.einsum("mr,rk->mk", u, d["a"][i])
                da[i], db[i] = torch.einsum("mr,mk->rk", u, x), torch.einsum("mr,mn->rn", v, gy)
        return {"y": y, "dx": dx, "da": da, "db": db} if case["train"] else {"y": y}
    p = case["p"]
    factor = None
    if p > 0:
        factor = _exact_kept(case["rows"], case["cols"], p, s["seed"], s["call"]).double() / (1.0 - p)
    h = d["x"] if factor is None else d["x"] * factor
    if case["residual"]:
        h = h + d["residual"]
    if case["op"] == "dropout":
        return {"y": h, "dx": d["gy"] * factor} if case["train"] else {"y": h}
    var, mu = torch.var_mean(h, dim=1, correction=0, keepdim=True)
    std = (var + EPS).sqrt()
    unit = (h - mu) / std
    out = {"y": unit * d["weight"] + d["bias"]}
    if case["residual"]:
        out["h"] = h
    if case["train"]:
        g = d["gy"] * d["weight"]
        cols = case["cols"]
        dh = (cols * g - g.sum(1, keepdim=True) - unit * (g * unit).sum(1, keepdim=True)) / (cols * std)
        if case["residual"]:
            dh = dh + d["gh"]
            out["dresidual"] = dh
        out["dx"] = dh if factor is None else dh * factor
        out["dweight"], out["dbias"] = (d["gy"] * unit).sum(0), d["gy"].sum(0)
    return out
