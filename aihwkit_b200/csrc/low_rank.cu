// Low-rank adapters of many requests beside a shared projection: the rows of request j get
//   y = base + v b[id_j],   v = scale[id_j] x a[id_j]^T,   a [adapters, rank, k], b [adapters, rank, n]
// and the gradients of a and b. With both factors stored rank first, the gradient of x,
// (scale gy b^T) a, is the same operator with the factors' places changed, and the gradients of a
// and b are the same sum over rows, u^T x.
//
// lowRankApplyKernel. The work is narrow: 2 rank operations per element of x and of y, so memory
// bounds it up to ranks of about 64. A block takes up to 64 (or 16) rows of one request through both
// products: x is read once, v stays in shared memory, y is written once; nothing but the saved v
// goes through memory between the two. Operands go from global memory straight into the fragments
// of mma.sync: a dot product may run in any order, so a thread takes 16 neighbouring bytes of a row as
// its share of k, and columns are dealt to the fragments so that a thread ends up with 32
// neighbouring bytes of y. No operand is used by two warps, so staging would only add traffic. Where rows
// are few, a cluster of blocks shares a row tile: each takes a share of k, the partial v are added
// through distributed shared memory in rank order, and each block takes a share of the columns.
// Products: bf16 x bf16 and fp16 x fp16 are exact in the fp32 sum; fp32 factors (v, and x, a, b of
// fp32 calls) are split into two TF32 parts, hi + lo, and multiplied as hi hi + lo hi + hi lo, which leaves
// 2^-22 of a product out.
//
// lowRankGradKernel. grad[id] = sum over the rows of id of u^T x: a warp holds rank x 64 (or 32)
// columns in fragments and walks a chunk of rows of one request; chunks' partial sums go through memory
// and are added in the order of the rows (no atomics).
#include "digital.cuh"

#include <algorithm>

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace ab200 {

namespace {

// ---- segments ---------------------------------------------------------------------------------
// Rows are cut at the borders of the requests and then into tiles of 2^shift rows. With the
// borders c(0) = 0, c(1..n+1) = starts, c(n+2) = rows, segment j owns the tile slots from
// (c(j) >> shift) + j on: at least as many as it has tiles, so the slot of a tile needs no sum over
// the requests before it, and (rows >> shift) + n + 2 slots are enough. Surplus slots are empty.
struct Segments {
  const int *starts, *ids;
  int n, rows, adapters, shift;
};
struct RowTile {
  int row0, rows, id; // id < 0: no adapter
};
__device__ __forceinline__ int border(const Segments &s, int j) {
  return j == 0 ? 0 : j == s.n + 2 ? s.rows : min(max(s.starts[j - 1], 0), s.rows);
}
__device__ __forceinline__ RowTile findTile(const Segments &s, int slot) {
  RowTile t;
  int seg = slot;
  if (s.starts == nullptr) {
    t.row0 = slot; // one row each
    t.rows = slot < s.rows ? 1 : 0;
  } else {
    // the last segment whose first slot is not behind this one; every warp searches, 32 probes at a time
    const int lane = threadIdx.x & 31;
    int lo = 0, cnt = s.n + 2;
    while (cnt > 1) {
      const int step = (cnt + 31) / 32;
      const int j = lane * step;
      const bool le = j < cnt && (border(s, lo + j) >> s.shift) + lo + j <= slot;
      const unsigned hit = __ballot_sync(0xffffffffu, le);
      const int last = hit ? 31 - __clz(hit) : 0;
      lo += last * step;
      cnt = min(step, cnt - last * step);
    }
    const int begin = border(s, lo), end = border(s, lo + 1);
    const long long row0 = begin + ((long long)(slot - (begin >> s.shift) - lo) << s.shift);
    t.rows = row0 < begin ? 0 : (int)max(0LL, min((long long)end - row0, 1LL << s.shift));
    t.row0 = t.rows > 0 ? (int)row0 : 0;
    seg = lo - 1;
  }
  t.id = t.rows > 0 && seg >= 0 && seg < s.n ? s.ids[seg] : -1;
  if (t.id >= s.adapters) {
    t.id = -1;
  }
  return t;
}
long long segmentSlots(const LowRankRows &s, int shift) {
  return s.starts ? (s.rows >> shift) + s.segments + 2 : s.rows;
}

// ---- fragments --------------------------------------------------------------------------------
__device__ __forceinline__ void mmaTf32(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},"
               "{%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T>
__device__ __forceinline__ void mma16(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},"
               "{%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16<__half>(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},"
               "{%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// fp32 = hi + lo, hi the nearest value of 11 bits, lo the exact rest (12 bits at most, of which the
// multiplier reads 11)
__device__ __forceinline__ void split(float v, uint32_t &hi, uint32_t &lo) {
  hi = (__float_as_uint(v) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(v - __uint_as_float(hi));
}

// 16 bytes of a row: eight 16-bit or four fp32 neighbours; elements past the end read as zero
template <typename T, bool VEC>
__device__ __forceinline__ uint4 load16B(const T *p, int col, int cols) {
  constexpr int E = 16 / sizeof(T);
  uint4 q = make_uint4(0, 0, 0, 0);
  if (VEC) {
    if (col < cols) {
      q = *reinterpret_cast<const uint4 *>(p + col);
    }
  } else {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < E; i++) {
      if (col + i < cols) {
        if (sizeof(T) == 4) {
          w[i & 3] = reinterpret_cast<const uint32_t *>(p)[col + i];
        } else {
          w[i >> 1] |= (uint32_t) reinterpret_cast<const uint16_t *>(p)[col + i] << (16 * (i & 1));
        }
      }
    }
    q = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return q;
}
// element i of 16 bytes, as fp32 (exact in TF32 for 16-bit types)
template <typename T> __device__ __forceinline__ float elemOf(const uint4 &q, int i) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(w[i & 3]);
  } else {
    const float2 f = unpack2<T>(w[i >> 1]);
    return (i & 1) ? f.y : f.x;
  }
}
__device__ __forceinline__ uint32_t wordOf(const uint4 &q, int i) {
  return i == 0 ? q.x : i == 1 ? q.y : i == 2 ? q.z : q.w;
}

// c += a b for one k-share of 16 bytes a row: x rows g and g + 8, factor row g
template <typename T>
__device__ __forceinline__ void mmaShare(float c[4], const uint4 &xg, const uint4 &xg8, const uint4 &f) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      uint32_t ah[4], al[4], bh[2], bl[2];
      split(__uint_as_float(wordOf(xg, 2 * h)), ah[0], al[0]);
      split(__uint_as_float(wordOf(xg8, 2 * h)), ah[1], al[1]);
      split(__uint_as_float(wordOf(xg, 2 * h + 1)), ah[2], al[2]);
      split(__uint_as_float(wordOf(xg8, 2 * h + 1)), ah[3], al[3]);
      split(__uint_as_float(wordOf(f, 2 * h)), bh[0], bl[0]);
      split(__uint_as_float(wordOf(f, 2 * h + 1)), bh[1], bl[1]);
      mmaTf32(c, al, bh[0], bh[1]);
      mmaTf32(c, ah, bl[0], bl[1]);
      mmaTf32(c, ah, bh[0], bh[1]);
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const uint32_t a[4] = {wordOf(xg, 2 * h), wordOf(xg8, 2 * h), wordOf(xg, 2 * h + 1), wordOf(xg8, 2 * h + 1)};
      mma16<T>(c, a, wordOf(f, 2 * h), wordOf(f, 2 * h + 1));
    }
  }
}
// c[j] += (hi + lo) b for the neighbouring columns j of one thread: b0 from row t of the factor, b1
// from row t + 4
template <typename T, int NJ>
__device__ __forceinline__ void mmaColumns(float (*c)[4], const uint32_t hi[4], const uint32_t lo[4], const uint4 &b0,
                                           const uint4 &b1) {
#pragma unroll
  for (int j = 0; j < NJ; j++) {
    const float f0 = elemOf<T>(b0, j), f1 = elemOf<T>(b1, j);
    if constexpr (sizeof(T) == 4) {
      uint32_t h0, l0, h1, l1;
      split(f0, h0, l0);
      split(f1, h1, l1);
      mmaTf32(c[j], lo, h0, h1);
      mmaTf32(c[j], hi, l0, l1);
      mmaTf32(c[j], hi, h0, h1);
    } else {
      mmaTf32(c[j], lo, __float_as_uint(f0), __float_as_uint(f1));
      mmaTf32(c[j], hi, __float_as_uint(f0), __float_as_uint(f1));
    }
  }
}

// 32 neighbouring bytes of a row: 16 16-bit or eight fp32 elements
template <typename T, bool VEC>
__device__ __forceinline__ void load32Bytes(const T *row, int col, int cols, uint4 q[2]) {
  q[0] = load16B<T, VEC>(row, col, cols);
  q[1] = load16B<T, VEC>(row, col + 16 / (int)sizeof(T), cols);
}
template <typename T, bool VEC>
__device__ __forceinline__ void store32Bytes(T *row, int col, int cols, const float *v) {
  constexpr int E = 32 / sizeof(T);
  if (VEC) {
    if (col < cols) {
      if constexpr (sizeof(T) == 4) {
        store32B(reinterpret_cast<float *>(row) + col, v);
      } else {
#pragma unroll
        for (int h = 0; h < 2; h++) {
          uint4 q;
          q.x = pack2<T>(v[8 * h], v[8 * h + 1]);
          q.y = pack2<T>(v[8 * h + 2], v[8 * h + 3]);
          q.z = pack2<T>(v[8 * h + 4], v[8 * h + 5]);
          q.w = pack2<T>(v[8 * h + 6], v[8 * h + 7]);
          reinterpret_cast<uint4 *>(row + col)[h] = q;
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; i++) {
      if (col + i < cols) {
        row[col + i] = Elem<T>::put(v[i]);
      }
    }
  }
}

// ---- apply ------------------------------------------------------------------------------------
struct Apply {
  Segments seg;
  const void *x, *base, *a, *b;
  void *y;
  const float *scale;
  float *v;
  long long x_ld, base_ld, y_ld;
  int k, n, rank;
  int cluster;
};

constexpr int kApplyThreads = 256;

// MT fragments of 16 rows per warp, WM warps over the rows, the other warps share k and the columns;
// ranks go through the first product 8 * NT at a time
template <typename T, bool VEC, int MT, int WM, int NT>
__global__ void __launch_bounds__(kApplyThreads, 2) lowRankApplyKernel(Apply p) {
  constexpr int WARPS = kApplyThreads / 32, WK = WARPS / WM, TM = 16 * MT * WM, RC = 8 * NT, RS = RC + 4;
  constexpr int E = 16 / sizeof(T), KS = 4 * E; // elements of k per thread, per fragment row and step
  constexpr int NJ = E, UC = 8 * NJ;            // columns per thread of a factor, per unit of a warp
  extern __shared__ float smem[];
  pdlEnter();
  const int part = p.cluster > 1 ? blockIdx.x % p.cluster : 0;
  const RowTile tile = findTile(p.seg, blockIdx.x / p.cluster);
  if (tile.rows <= 0) {
    return; // the whole cluster has the same tile
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int wm = warp / WK, wk = warp % WK;
  const int units = (p.n + UC - 1) / UC, units_per = (units + p.cluster - 1) / p.cluster;
  const int u_begin = part * units_per, u_end = min(units, u_begin + units_per);
  int row[MT][2]; // rows of this thread's fragments, -1 past the tile
#pragma unroll
  for (int i = 0; i < MT; i++) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int r = wm * 16 * MT + i * 16 + h * 8 + g;
      row[i][h] = r < tile.rows ? tile.row0 + r : -1;
    }
  }
  if (tile.id < 0) {
    // no adapter: y is base (nothing to do where they are the same memory) or zero
    if (p.y == nullptr || p.y == p.base) {
      return;
    }
    for (int u = u_begin + wk; u < u_end; u += WK) {
      const int col = u * UC + 2 * NJ * t;
#pragma unroll
      for (int i = 0; i < MT; i++) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
          if (row[i][h] >= 0) {
            uint4 q[2] = {};
            if (p.base) {
              load32Bytes<T, VEC>((const T *)p.base + row[i][h] * p.base_ld, col, p.n, q);
            }
            float o[2 * NJ];
#pragma unroll
            for (int j = 0; j < 2 * NJ; j++) {
              o[j] = elemOf<T>(q[j / NJ], j % NJ);
            }
            store32Bytes<T, VEC>((T *)p.y + row[i][h] * p.y_ld, col, p.n, o);
          }
        }
      }
    }
    return;
  }
  const int r_pad = (p.rank + 7) & ~7, vs = r_pad + 4;
  float *mine = smem;             // [TM][vs]: this block's share of v
  float *red = smem + TM * vs;    // [WK][TM][RS] while the warps' shares are added
  float *full = p.cluster > 1 ? red : mine; // [TM][vs]: v of the tile
  const float scale = p.scale[tile.id];
  const T *fa = (const T *)p.a + (long long)tile.id * p.rank * p.k;
  const T *fb = (const T *)p.b + (long long)tile.id * p.rank * p.n;

  // v = x a^T: steps of KS along k are dealt to the blocks of the cluster and to the warps in turn
  const int steps = (p.k + KS - 1) / KS, steps_per = (steps + p.cluster - 1) / p.cluster;
  const int s_end = min(steps, (part + 1) * steps_per);
  for (int r0 = 0; r0 < p.rank; r0 += RC) {
    float acc[MT][NT][4];
#pragma unroll
    for (int i = 0; i < MT; i++) {
#pragma unroll
      for (int j = 0; j < NT; j++) {
        acc[i][j][0] = acc[i][j][1] = acc[i][j][2] = acc[i][j][3] = 0.0f;
      }
    }
#pragma unroll 2
    for (int s = part * steps_per + wk; s < s_end; s += WK) {
      const int k0 = s * KS + t * E;
      uint4 x[MT][2], f[NT];
#pragma unroll
      for (int i = 0; i < MT; i++) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
          x[i][h] = row[i][h] >= 0 ? load16B<T, VEC>((const T *)p.x + row[i][h] * p.x_ld, k0, p.k)
                                   : make_uint4(0, 0, 0, 0);
        }
      }
#pragma unroll
      for (int j = 0; j < NT; j++) {
        const int r = r0 + j * 8 + g;
        f[j] = r < p.rank ? load16B<T, VEC>(fa + (long long)r * p.k, k0, p.k) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int j = 0; j < NT; j++) {
#pragma unroll
        for (int i = 0; i < MT; i++) {
          mmaShare<T>(acc[i][j], x[i][0], x[i][1], f[j]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < MT; i++) {
#pragma unroll
      for (int j = 0; j < NT; j++) {
        float *d = red + (wk * TM + wm * 16 * MT + i * 16 + g) * RS + j * 8 + 2 * t;
        *reinterpret_cast<float2 *>(d) = make_float2(acc[i][j][0], acc[i][j][1]);
        *reinterpret_cast<float2 *>(d + 8 * RS) = make_float2(acc[i][j][2], acc[i][j][3]);
      }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < TM * RC; e += kApplyThreads) {
      const int r = e / RC, c = e % RC;
      if (r0 + c < r_pad) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < WK; w++) {
          sum += red[(w * TM + r) * RS + c];
        }
        mine[r * vs + r0 + c] = p.cluster > 1 ? sum : sum * scale;
      }
    }
    __syncthreads();
  }
  if (p.cluster > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int e = threadIdx.x; e < TM * r_pad; e += kApplyThreads) {
      const int o = (e / r_pad) * vs + e % r_pad;
      float sum = 0.0f;
      for (int q = 0; q < p.cluster; q++) {
        sum += cluster.map_shared_rank(mine, q)[o];
      }
      full[o] = sum * scale;
    }
    cluster.sync(); // no block leaves, and none reads `full`, before all have read the shares
  }
  if (p.v != nullptr && part == 0) {
    for (int e = threadIdx.x; e < tile.rows * p.rank; e += kApplyThreads) {
      p.v[(long long)tile.row0 * p.rank + e] = full[(e / p.rank) * vs + e % p.rank];
    }
  }
  if (p.y == nullptr) {
    return;
  }

  // y = base + v b: units of UC columns are dealt to the blocks of the cluster and to the warps
  const float *vrow = full + (wm * 16 * MT + g) * vs + t;
  for (int u = u_begin + wk; u < u_end; u += WK) {
    const int col = u * UC + 2 * NJ * t;
    uint4 old[MT][2][2] = {};
    if (p.base) {
#pragma unroll
      for (int i = 0; i < MT; i++) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
          if (row[i][h] >= 0) {
            load32Bytes<T, VEC>((const T *)p.base + row[i][h] * p.base_ld, col, p.n, old[i][h]);
          }
        }
      }
    }
    float acc[MT][NJ][4];
#pragma unroll
    for (int i = 0; i < MT; i++) {
#pragma unroll
      for (int j = 0; j < NJ; j++) {
        acc[i][j][0] = acc[i][j][1] = acc[i][j][2] = acc[i][j][3] = 0.0f;
      }
    }
    const int fcol = u * UC + NJ * g;
#pragma unroll 2
    for (int r = 0; r < r_pad; r += 8) {
      const uint4 none = make_uint4(0, 0, 0, 0);
      const uint4 b0 = r + t < p.rank ? load16B<T, VEC>(fb + (long long)(r + t) * p.n, fcol, p.n) : none;
      const uint4 b1 = r + t + 4 < p.rank ? load16B<T, VEC>(fb + (long long)(r + t + 4) * p.n, fcol, p.n) : none;
#pragma unroll
      for (int i = 0; i < MT; i++) {
        uint32_t hi[4], lo[4];
        const float *v = vrow + i * 16 * vs + r;
        split(v[0], hi[0], lo[0]);
        split(v[8 * vs], hi[1], lo[1]);
        split(v[4], hi[2], lo[2]);
        split(v[8 * vs + 4], hi[3], lo[3]);
        mmaColumns<T, NJ>(acc[i], hi, lo, b0, b1);
      }
    }
#pragma unroll
    for (int i = 0; i < MT; i++) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        if (row[i][h] >= 0) {
          float o[2 * NJ];
#pragma unroll
          for (int j = 0; j < NJ; j++) {
            o[j] = acc[i][j][2 * h] + elemOf<T>(old[i][h][0], j);
            o[NJ + j] = acc[i][j][2 * h + 1] + elemOf<T>(old[i][h][1], j);
          }
          store32Bytes<T, VEC>((T *)p.y + row[i][h] * p.y_ld, col, p.n, o);
        }
      }
    }
  }
}

template <typename T, bool VEC, int MT, int WM, int NT>
void launchApply(Apply p, long long slots, cudaStream_t stream) {
  constexpr int WK = kApplyThreads / 32 / WM, TM = 16 * MT * WM;
  const int vs = ((p.rank + 7) & ~7) + 4;
  const size_t smem = sizeof(float) * ((size_t)TM * vs + std::max((size_t)WK * TM * (8 * NT + 4), (size_t)TM * vs));
  auto kernel = lowRankApplyKernel<T, VEC, MT, WM, NT>;
  if (smem > 48 * 1024) {
    AB200_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(slots * p.cluster));
  cfg.blockDim = dim3(kApplyThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdlEnabled() ? 2 : 1;
  AB200_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
  AB200_LAUNCH_CHECK();
}
template <typename T, bool VEC, int MT, int WM> void dispatchRank(const Apply &p, long long slots, cudaStream_t st) {
  if (p.rank <= 8) {
    launchApply<T, VEC, MT, WM, 1>(p, slots, st);
  } else if (p.rank <= 16) {
    launchApply<T, VEC, MT, WM, 2>(p, slots, st);
  } else if (p.rank <= 32) {
    launchApply<T, VEC, MT, WM, 4>(p, slots, st);
  } else {
    launchApply<T, VEC, MT, WM, 8>(p, slots, st);
  }
}
template <typename T> void dispatchApply(Apply p, const LowRankRows &seg, bool vec, cudaStream_t st) {
  // Requests of 16 rows and fewer on average (decoding) take tiles of 16 rows, longer ones of 64.
  const bool small = seg.starts == nullptr || seg.rows <= 16LL * seg.segments;
  p.seg.shift = small ? 4 : 6;
  const long long slots = segmentSlots(seg, p.seg.shift);
  // Blocks that share a tile: as many as it takes to occupy the multiprocessors, eight at most
  const int sms = digitalSmCount();
  p.cluster = 1;
  while (p.cluster < 8 && slots * p.cluster < sms) {
    p.cluster *= 2;
  }
  if (small) {
    vec ? dispatchRank<T, true, 1, 1>(p, slots, st) : dispatchRank<T, false, 1, 1>(p, slots, st);
  } else {
    vec ? dispatchRank<T, true, 2, 2>(p, slots, st) : dispatchRank<T, false, 2, 2>(p, slots, st);
  }
}

// ---- gradients of the factors -----------------------------------------------------------------
struct Grad {
  Segments seg;
  const void *x[2];
  long long x_ld[2];
  const float *u[2];
  float *partial[2]; // [slots][rank][width]
  int *slot_id;      // [slots]
  int width[2];
  int rank, rank_passes;
};

constexpr int kGradWarps = 4;

template <typename T, bool VEC, int RT>
__global__ void __launch_bounds__(kGradWarps * 32) lowRankGradKernel(Grad p) {
  constexpr int NJ = 16 / sizeof(T), UC = 8 * NJ;
  pdlEnter();
  const int side = blockIdx.z / p.rank_passes, r0 = (blockIdx.z % p.rank_passes) * 16 * RT;
  const RowTile tile = findTile(p.seg, blockIdx.x);
  if (blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x == 0) {
    p.slot_id[blockIdx.x] = tile.rows > 0 ? tile.id : -1;
  }
  const int width = side ? p.width[1] : p.width[0];
  const long long ld = side ? p.x_ld[1] : p.x_ld[0];
  float *partial = side ? p.partial[1] : p.partial[0];
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int unit = blockIdx.y * kGradWarps + (threadIdx.x >> 5);
  if (tile.rows <= 0 || tile.id < 0 || partial == nullptr || unit * UC >= width) {
    return;
  }
  const T *x = (const T *)(side ? p.x[1] : p.x[0]) + tile.row0 * ld;
  const float *u = (side ? p.u[1] : p.u[0]) + (long long)tile.row0 * p.rank + r0;
  const int ranks = p.rank - r0, fcol = unit * UC + NJ * g;
  float acc[RT][NJ][4];
#pragma unroll
  for (int i = 0; i < RT; i++) {
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      acc[i][j][0] = acc[i][j][1] = acc[i][j][2] = acc[i][j][3] = 0.0f;
    }
  }
#pragma unroll 4
  for (int r = 0; r < tile.rows; r += 8) {
    const bool in0 = r + t < tile.rows, in1 = r + t + 4 < tile.rows;
    const uint4 none = make_uint4(0, 0, 0, 0);
    const uint4 x0 = in0 ? load16B<T, VEC>(x + (r + t) * ld, fcol, width) : none;
    const uint4 x1 = in1 ? load16B<T, VEC>(x + (r + t + 4) * ld, fcol, width) : none;
#pragma unroll
    for (int i = 0; i < RT; i++) {
      const float *u0 = u + (long long)(r + t) * p.rank + i * 16 + g, *u1 = u0 + 4 * p.rank;
      const bool lowr = i * 16 + g < ranks, highr = i * 16 + g + 8 < ranks;
      uint32_t hi[4], lo[4];
      split(in0 && lowr ? u0[0] : 0.0f, hi[0], lo[0]);
      split(in0 && highr ? u0[8] : 0.0f, hi[1], lo[1]);
      split(in1 && lowr ? u1[0] : 0.0f, hi[2], lo[2]);
      split(in1 && highr ? u1[8] : 0.0f, hi[3], lo[3]);
      mmaColumns<T, NJ>(acc[i], hi, lo, x0, x1);
    }
  }
  const int col = unit * UC + 2 * NJ * t;
  float *out = partial + ((long long)blockIdx.x * p.rank + r0) * width;
#pragma unroll
  for (int i = 0; i < RT; i++) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int r = i * 16 + h * 8 + g;
      if (r < ranks) {
#pragma unroll
        for (int j = 0; j < 2 * NJ; j++) {
          if (col + j < width) {
            out[(long long)r * width + col + j] = acc[i][j % NJ][2 * h + j / NJ];
          }
        }
      }
    }
  }
}

// grad[i] = sum of the partial sums of adapter i's chunks, in the order of the rows; zero without any
template <typename T>
__global__ void __launch_bounds__(256)
    lowRankJoinKernel(const int *__restrict__ slot_id, int slots, const float *__restrict__ p0,
                      const float *__restrict__ p1, T *g0, T *g1, long long elems0, long long elems1) {
  pdlEnter();
  const int side = blockIdx.z, i = blockIdx.y;
  const long long elems = side ? elems1 : elems0;
  const float *partial = side ? p1 : p0;
  T *grad = side ? g1 : g0;
  const long long e = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (grad == nullptr || e >= elems) {
    return;
  }
  float sum = 0.0f;
  for (int s = 0; s < slots; s++) {
    if (slot_id[s] == i) {
      sum += partial[s * elems + e];
    }
  }
  grad[i * elems + e] = Elem<T>::put(sum);
}

// rows per chunk: enough blocks for three per multiprocessor, between 32 and 2048 rows
int gradShift(const LowRankRows &s, int width0, int width1) {
  int shift = 11;
  const long long units = (width0 + width1 + 255) / 256;
  while (shift > 5 && units * (s.rows >> shift) < 3LL * digitalSmCount()) {
    shift--;
  }
  return shift;
}
long long gradSlots(const LowRankRows &s, int width0, int width1, int *shift) {
  *shift = gradShift(s, width0, width1);
  return segmentSlots(s, *shift);
}
long long idBytes(long long slots) { return (slots * 4 + 255) / 256 * 256; }

template <typename T, bool VEC> void launchGrad(Grad p, long long slots, cudaStream_t st) {
  const int widest = std::max(p.partial[0] ? p.width[0] : 0, p.partial[1] ? p.width[1] : 0);
  const int uc = 8 * (16 / (int)sizeof(T)) * kGradWarps;
  const int rt = p.rank <= 16 ? 1 : p.rank <= 32 ? 2 : 4;
  p.rank_passes = (p.rank + 16 * rt - 1) / (16 * rt);
  const dim3 grid((unsigned)slots, (unsigned)((widest + uc - 1) / uc), (unsigned)(2 * p.rank_passes));
  auto kernel = rt == 1 ? lowRankGradKernel<T, VEC, 1> : rt == 2 ? lowRankGradKernel<T, VEC, 2> : lowRankGradKernel<T, VEC, 4>;
  AB200_CUDA(launchChained(kernel, grid, dim3(kGradWarps * 32), 0, st, p));
  AB200_LAUNCH_CHECK();
}
template <typename T>
void gradOfType(const Grad &p, const LowRankGradArgs &a, long long slots, bool vec, cudaStream_t st) {
  if (slots > 0) {
    vec ? launchGrad<T, true>(p, slots, st) : launchGrad<T, false>(p, slots, st);
  }
  const long long e0 = (long long)a.rank * a.width[0], e1 = (long long)a.rank * a.width[1];
  const long long most = std::max(a.grad[0] ? e0 : 0, a.grad[1] ? e1 : 0);
  AB200_CUDA(launchChained(lowRankJoinKernel<T>, dim3((unsigned)((most + 255) / 256), (unsigned)a.adapters, 2), dim3(256),
                           0, st, (const int *)p.slot_id, (int)slots, (const float *)p.partial[0],
                           (const float *)p.partial[1], (T *)a.grad[0], (T *)a.grad[1], e0, e1));
  AB200_LAUNCH_CHECK();
}

bool rowsAlign(const void *p, long long ld, int width, int type) {
  const int size = type == DT_F32 ? 4 : 2;
  return p == nullptr || ((uintptr_t)p % 32 == 0 && ld * size % 32 == 0 && (long long)width * size % 32 == 0);
}

} // namespace

void lowRankApply(const LowRankArgs &a, cudaStream_t stream) {
  if (a.seg.rows <= 0) {
    return;
  }
  Apply p = {};
  p.seg = {a.seg.starts, a.seg.ids, a.seg.segments, (int)a.seg.rows, a.adapters, 0};
  p.x = a.x.p;
  p.x_ld = a.x.ld;
  p.base = a.base.p;
  p.base_ld = a.base.ld;
  p.y = a.y.p;
  p.y_ld = a.y.ld;
  p.a = a.a;
  p.b = a.b;
  p.scale = a.scale;
  p.v = a.v;
  p.k = a.k;
  p.n = a.n;
  p.rank = a.rank;
  const bool vec = rowsAlign(a.x.p, a.x.ld, a.k, a.type) && rowsAlign(a.base.p, a.base.ld, a.n, a.type) &&
                   rowsAlign(a.y.p, a.y.ld, a.n, a.type) && rowsAlign(a.a, a.k, a.k, a.type) &&
                   rowsAlign(a.b, a.n, a.n, a.type);
  switch (a.type) {
  case DT_F32: dispatchApply<float>(p, a.seg, vec, stream); break;
  case DT_F16: dispatchApply<__half>(p, a.seg, vec, stream); break;
  default: dispatchApply<__nv_bfloat16>(p, a.seg, vec, stream);
  }
}

long long lowRankGradWorkspace(long long rows, int segments, bool one_row_each, int width0, int width1, int rank) {
  int shift = 0;
  const int some = 0;
  const LowRankRows s = {one_row_each ? nullptr : &some, nullptr, segments, rows};
  const long long slots = rows > 0 ? gradSlots(s, width0, width1, &shift) : 0;
  return idBytes(slots) + slots * rank * ((long long)width0 + width1) * 4;
}

void lowRankGrad(const LowRankGradArgs &a, cudaStream_t stream) {
  if (!a.grad[0] && !a.grad[1]) {
    return;
  }
  int shift = 0;
  const int w0 = a.grad[0] ? a.width[0] : 0, w1 = a.grad[1] ? a.width[1] : 0;
  const long long slots = a.seg.rows > 0 ? gradSlots(a.seg, w0, w1, &shift) : 0;
  Grad p = {};
  p.seg = {a.seg.starts, a.seg.ids, a.seg.segments, (int)a.seg.rows, a.adapters, shift};
  bool vec = true;
  float *next = reinterpret_cast<float *>((char *)a.workspace + idBytes(slots));
  p.slot_id = (int *)a.workspace;
  for (int q = 0; q < 2; q++) {
    p.x[q] = a.x[q].p;
    p.x_ld[q] = a.x[q].ld;
    p.u[q] = a.u[q];
    p.width[q] = a.width[q];
    p.partial[q] = a.grad[q] ? next : nullptr;
    if (a.grad[q]) {
      next += slots * a.rank * a.width[q];
      vec = vec && rowsAlign(a.x[q].p, a.x[q].ld, a.width[q], a.type);
    }
  }
  p.rank = a.rank;
  switch (a.type) {
  case DT_F32: gradOfType<float>(p, a, slots, vec, stream); break;
  case DT_F16: gradOfType<__half>(p, a, slots, vec, stream); break;
  default: gradOfType<__nv_bfloat16>(p, a, slots, vec, stream);
  }
}

} // namespace ab200
