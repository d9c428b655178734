"""The GPT-2-shaped model with low-rank adapters beside its analog layers: loss and gradients against the same model in plain
operations and 64 bits (perfect tiles), and the command's options."""

import json

import pytest
import torch
import torch.nn.functional as F

from aihwkit_b200 import gpt2_inference as G
from tests.test_digital_gpu import kept

pytestmark = pytest.mark.gpu


def small_model(monkeypatch, adapters=3, rank=4):
    from aihwkit_b200.rpu_base import devices as D

    def config(seed, max_tile=512, adapted=False):
        p = D.AnalogTileParameter()
        p.forward_io.is_perfect = p.backward_io.is_perfect = True
        p.update.pulse_type = D.PulseType.None_
        return p._config(max_tile, max_tile, D.IdealResistiveDeviceParameter(), seed=seed)

    monkeypatch.setattr(G, "inference_config", config)
    monkeypatch.setattr(G, "VOCAB", 211)
    model = G.AnalogGPT2(2, d_model=64, n_head=2, seed=3, adapters=adapters, rank=rank)
    g = torch.Generator(device="cuda").manual_seed(1)
    for lin in (lin for blk in model.blocks for lin in blk.linears()):
        with torch.no_grad():
            lin.adapters.b.normal_(0, 0.2, generator=g)
            lin.adapters.scale.uniform_(0.5, 1.5, generator=g)
    for t in model.trained():
        if t.dim() == 1:
            t.add_(torch.randn(t.shape, device="cuda", generator=g) * 0.1)
    return model


def plain_loss(model, leaves, ids, targets, adapter_ids, p, seed):
    """The same in 64 bits; ``leaves`` are the doubles of ``model.trained()``, in its order."""
    it = iter(leaves)
    pairs = [[(next(it), next(it)) for _ in blk.linears()] for blk in model.blocks]
    norms = [[next(it) for _ in range(4)] for _ in model.blocks] + [[next(it), next(it)]]
    b, s = ids.shape
    d = model.d_model
    call = [0]

    def linear(lin, ab, x):
        y = x @ lin.array.get_weights().cuda().double().t()
        a, bb = ab
        sc = lin.adapters.scale.double()[adapter_ids]
        return y + sc[:, None, None] * torch.einsum("bsr,brn->bsn", torch.einsum("bsk,brk->bsr", x, a[adapter_ids]), bb[adapter_ids])

    def drop(x):
        keep = kept(b * s, d, p, seed, call[0]).reshape(b, s, d)
        call[0] += 1
        return torch.where(keep, x / (1 - p), 0.0)

    h = (model.wte[ids] + model.wpe[:s]).double()
    for i, blk in enumerate(model.blocks):
        a = F.layer_norm(h, (d,), norms[i][0], norms[i][1])
        q, k, v = linear(blk.qkv, pairs[i][0], a).split(d, dim=-1)
        q, k, v = (t.reshape(b, s, blk.n_head, -1).transpose(1, 2) for t in (q, k, v))
        w = (q @ k.transpose(-1, -2)) / (d // blk.n_head) ** 0.5
        w = w.masked_fill(torch.ones(s, s, dtype=torch.bool, device="cuda").triu(1), float("-inf")).softmax(-1)
        h = h + drop(linear(blk.proj, pairs[i][1], (w @ v).transpose(1, 2).reshape(b, s, d)))
        a = F.layer_norm(h, (d,), norms[i][2], norms[i][3])
        h = h + drop(linear(blk.fc_out, pairs[i][3], F.gelu(linear(blk.fc, pairs[i][2], a))))
    h = F.layer_norm(h, (d,), *norms[-1])
    return F.cross_entropy(h.reshape(-1, d) @ model.wte.double().t(), targets.reshape(-1))


@pytest.mark.parametrize("p", [0.0, 0.2])
def test_loss_and_gradients(monkeypatch, p):
    model = small_model(monkeypatch)
    g = torch.Generator().manual_seed(2)
    ids = torch.randint(0, 211, (4, 37), generator=g).cuda()
    targets = torch.randint(0, 211, (4, 37), generator=g).cuda()
    adapter_ids = torch.tensor([2, 0, 2, 1], device="cuda")
    weights = model.trained()
    for t in weights:
        t.requires_grad_()
    loss = model.loss(ids, targets, G.Adaptation(adapter_ids, 37, p, seed=9))
    grads = torch.autograd.grad(loss, weights)
    leaves = [t.detach().double().requires_grad_() for t in weights]
    want = plain_loss(model, leaves, ids, targets, adapter_ids, p, 9)
    want_grads = torch.autograd.grad(want, leaves)
    # about forty fp32 operators in a row, each off by at most some 64 roundings of 2^-24
    tol = 40 * 64 * 2.0 ** -24
    assert abs(float(loss.detach()) - float(want.detach())) <= tol * float(want.detach())
    for got, ref in zip(grads, want_grads):
        assert float((got.double() - ref).norm()) <= tol * float(ref.norm())
    with torch.no_grad():  # adapters in place on the tiles' results, without a graph
        again = model.loss(ids, targets, G.Adaptation(adapter_ids, 37, p, seed=9))
    assert abs(float(again) - float(want.detach())) <= tol * float(want.detach())


def test_command_with_adapters(capsys):
    G.main(["--layers", "1", "--batch", "2", "--seq", "64", "--steps", "1", "--warmup", "1", "--adapters", "2", "--rank", "8",
            "--adapt-steps", "2"])
    out = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    assert out["adapters"] == {"count": 2, "rank": 8} and out["value"] > 0
    assert out["adaptation"]["steps"] == 2 and all(0 < v < 100 for v in out["adaptation"]["losses"])
    with pytest.raises(SystemExit):
        G.main(["--adapt-steps", "1"])


def test_adapters_beside_sharded_tiles_are_refused():
    with pytest.raises(RuntimeError, match="adapters are built for layers whose tiles are all on one GPU"):
        G.AnalogLinear(64, 64, 0, 1, torch.Generator().manual_seed(0), shard_tiles=True, adapters=2)
