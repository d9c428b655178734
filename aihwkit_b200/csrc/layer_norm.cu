// Layer norm, forward and backward, with the residual sum and the dropout in front of it:
//   h = residual + drop(x);  mu = mean h;  s = (mean (h - mu)^2 + eps)^-1/2;  y = (h - mu) s w + b
//   t = gy w;  u = (h - mu) s;  dh = s (t - mean t - u mean(t u)) + gh;  dx = drop(dh)
//   dw = sum over rows of gy u;  db = sum over rows of gy
// The backward pass sums h again from x and the residual rather than read the rounded one: an
// error of 2^-9 (bf16) of h would go straight into the fp32 sums of dw.
// Both passes are bound by memory, and next to it by instructions where 16-bit rows are dropped (Philox). A row is read
// once and stays in registers between its two sums (the squares are summed about the mean, so an offset of the
// row costs no digits). Rows of up to four spans of 256 columns (the backward pass: two) have a warp each (WIDE
// false, four rows to a block), longer ones a block.
// Measured: forward 16384 x 768 fp32 with residual 32.6 us (6.2 TB/s), 8192 x 4096 bf16 with residual and dropout 52
// us (5.2 TB/s), its backward pass 87 us (4.6 TB/s) and the sums over its blocks 6 us.
// Means, sums and gradients of the parameters are held in fp32; y and h are rounded once, from the
// unrounded sum.
#include "digital.cuh"

#include <algorithm>

namespace ab200 {

namespace {

constexpr int kRowThreads = 128; // of blocks whose warps have rows of their own

struct NormShape {
  long long rows;
  int cols;
  int spans;         // of 256 columns
  int per_warp;      // of them
  int warps_per_row; // warp w of a row has the spans w, w + warps_per_row, ...
  int rows_per_block;
  float inv_cols;
};

__device__ __forceinline__ float warpSum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  return v;
}
// sum over the warps of a row (at most 32); `red` has a slot per warp, used in turn so that one
// barrier per sum is enough
template <bool WIDE> __device__ __forceinline__ float rowSum(float v, int warps, float *red) {
  v = warpSum(v);
  if (WIDE) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) {
      red[threadIdx.x >> 5] = v;
    }
    __syncthreads();
    v = warpSum(lane < warps ? red[lane] : 0.0f);
  }
  return v;
}
template <bool WIDE> __device__ __forceinline__ float2 rowSum2(float a, float b, int warps, float2 *red) {
  a = warpSum(a);
  b = warpSum(b);
  if (WIDE) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) {
      red[threadIdx.x >> 5] = make_float2(a, b);
    }
    __syncthreads();
    const float2 t = lane < warps ? red[lane] : make_float2(0.0f, 0.0f);
    a = warpSum(t.x);
    b = warpSum(t.y);
  }
  return make_float2(a, b);
}

// parameters are read per row, from L1 after the first row of an SM
template <bool VEC>
__device__ __forceinline__ void loadParam(const void *p, int w_type, float none, int span, int lane, int cols,
                                          float v[8]) {
  if (p == nullptr) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      v[i] = none;
    }
    return;
  }
  if (w_type == DT_F32) {
    Raw8<float, VEC> r;
    r.load((const float *)p, span, lane, cols);
    r.get(v);
  } else if (w_type == DT_F16) {
    Raw8<__half, VEC> r;
    r.load((const __half *)p, span, lane, cols);
    r.get(v);
  } else {
    Raw8<__nv_bfloat16, VEC> r;
    r.load((const __nv_bfloat16 *)p, span, lane, cols);
    r.get(v);
  }
}

// The span of x behind the dropout. 16-bit rows are masked as they came, in pairs.
template <typename T, bool VEC>
__device__ __forceinline__ Kept dropped(const DropKey &key, long long row, int span, int lane, int cols, Raw8<T, VEC> &raw,
                                        float v[8]) {
  const Kept kept = keepOfSpan<VEC>(key, row, span, lane, cols);
  if constexpr (VEC && sizeof(T) == 2) {
    uint32_t m[4];
    pairMasks(kept, m);
    raw.mask(m);
    raw.get(v);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      v[i] *= key.scale;
    }
  } else {
    raw.get(v);
    dropSpan(key, kept, v);
  }
  return kept;
}

struct NormFwd {
  const void *x, *res, *w, *b;
  void *y, *h;
  float *mean, *rstd;
  long long x_ld, res_ld, y_ld, h_ld;
  int w_type;
  float eps;
  int drop;
};

template <typename T, bool VEC, bool WIDE, int NS>
__global__ void __launch_bounds__(WIDE ? 512 : kRowThreads)
    normForwardKernel(NormFwd a, NormShape sh, DropKey key) {
  pdlEnter();
  __shared__ float red[2][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int w0 = WIDE ? warp : 0;
  const long long row = (long long)blockIdx.x * sh.rows_per_block + (WIDE ? 0 : warp);
  if (row >= sh.rows) {
    return; // only whole warps of rows of their own
  }
  const T *xr = (const T *)a.x + row * a.x_ld;
  float v[NS][8];
  {
    Raw8<T, VEC> rx[NS], rr[NS];
#pragma unroll
    for (int s = 0; s < NS; s++) {
      rx[s].load(xr, w0 + s * sh.warps_per_row, lane, sh.cols);
    }
    if (a.res) {
      const T *rrow = (const T *)a.res + row * a.res_ld;
#pragma unroll
      for (int s = 0; s < NS; s++) {
        rr[s].load(rrow, w0 + s * sh.warps_per_row, lane, sh.cols);
      }
    }
#pragma unroll
    for (int s = 0; s < NS; s++) {
      const int span = w0 + s * sh.warps_per_row;
      if (a.drop) {
        dropped<T, VEC>(key, row, span, lane, sh.cols, rx[s], v[s]);
      } else {
        rx[s].get(v[s]);
      }
      if (a.res) {
        float r[8];
        rr[s].get(r);
#pragma unroll
        for (int i = 0; i < 8; i++) {
          v[s][i] += r[i];
        }
      }
    }
  }
  float sum = 0.0f;
#pragma unroll
  for (int s = 0; s < NS; s++) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      sum += v[s][i]; // columns past the end hold zeros
    }
  }
  if (a.h) {
#pragma unroll
    for (int s = 0; s < NS; s++) {
      storeSpan<T, VEC>((T *)a.h + row * a.h_ld, w0 + s * sh.warps_per_row, lane, sh.cols, v[s]);
    }
  }
  const float mean = rowSum<WIDE>(sum, sh.warps_per_row, red[0]) * sh.inv_cols;
  float sq = 0.0f;
#pragma unroll
  for (int s = 0; s < NS; s++) {
    const int span = w0 + s * sh.warps_per_row;
    const bool all = VEC && Span<VEC>::col(span, lane, 0) < sh.cols; // of a lane's eight neighbours
#pragma unroll
    for (int i = 0; i < 8; i++) {
      v[s][i] -= mean;
      const bool in = VEC ? all : Span<VEC>::col(span, lane, i) < sh.cols;
      sq = in ? fmaf(v[s][i], v[s][i], sq) : sq;
    }
  }
  const float var = rowSum<WIDE>(sq, sh.warps_per_row, red[1]) * sh.inv_cols;
  const float rstd = rsqrtf(var + a.eps);
  if (a.mean != nullptr && lane == 0 && w0 == 0) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
#pragma unroll
  for (int s = 0; s < NS; s++) {
    const int span = w0 + s * sh.warps_per_row;
    float w[8], b[8];
    loadParam<VEC>(a.w, a.w_type, 1.0f, span, lane, sh.cols, w);
    loadParam<VEC>(a.b, a.w_type, 0.0f, span, lane, sh.cols, b);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      w[i] = fmaf(v[s][i] * rstd, w[i], b[i]);
    }
    storeSpan<T, VEC>((T *)a.y + row * a.y_ld, span, lane, sh.cols, w);
  }
}

struct NormBwd {
  const void *gy, *gh, *x, *res, *w;
  void *dh, *dx;
  const float *mean, *rstd;
  float *partial; // [blocks][2][cols]
  long long gy_ld, gh_ld, x_ld, res_ld, dh_ld, dx_ld;
  int w_type;
  int drop; // x is dropped before the sum
};

// 16-bit rows are fetched ahead by blocks of few warps on long rows, where the registers leave room for no third
// block; fp32 ones of four tensors would not fit shared memory at 8192 columns
template <typename T> constexpr bool normAhead(bool vec, bool wide, int ns) {
  return vec && wide && ns == 2 && sizeof(T) == 2;
}
__host__ __device__ inline int normTensors(const NormBwd &a) { return 2 + (a.res ? 1 : 0) + (a.gh ? 1 : 0); }

// Blocks walk over the rows with a fixed stride and keep the sums of the parameters' gradients of
// their columns in registers; a second kernel adds the blocks' sums in order, so the result does
// not depend on which block ran when.
template <typename T, bool VEC, bool WIDE, int NS>
__global__ void __launch_bounds__(WIDE ? 512 : kRowThreads, WIDE && NS == 1 ? 2 : 1)
    normBackwardKernel(NormBwd a, NormShape sh, DropKey key) {
  constexpr bool AHEAD = normAhead<T>(VEC, WIDE, NS);
  pdlEnter();
  __shared__ float2 red[2][32];
  // the rows ahead; where a block has several rows, [2][cols] for its sums at the end
  extern __shared__ __align__(16) float dynamic[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int w0 = WIDE ? warp : 0, ws = sh.warps_per_row;
  float dw[NS][8], db[NS][8];
#pragma unroll
  for (int s = 0; s < NS; s++) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      dw[s][i] = db[s][i] = 0.0f;
    }
  }
  const long long stride = (long long)gridDim.x * sh.rows_per_block;
  const int slot_res = 2, slot_gh = a.res ? 3 : 2;
  const RowRing<T, NS> ring(dynamic, normTensors(a));
  const auto fetch = [&](long long row, int stage) {
    if (row < sh.rows) {
#pragma unroll
      for (int s = 0; s < NS; s++) {
        const int span = w0 + s * ws;
        ring.issue(stage, 0, s, (const T *)a.x + row * a.x_ld, span, lane, sh.cols);
        ring.issue(stage, 1, s, (const T *)a.gy + row * a.gy_ld, span, lane, sh.cols);
        if (a.res) {
          ring.issue(stage, slot_res, s, (const T *)a.res + row * a.res_ld, span, lane, sh.cols);
        }
        if (a.gh) {
          ring.issue(stage, slot_gh, s, (const T *)a.gh + row * a.gh_ld, span, lane, sh.cols);
        }
      }
    }
    ring.commit();
  };
  long long row = (long long)blockIdx.x * sh.rows_per_block + (WIDE ? 0 : warp);
  if (AHEAD) {
    fetch(row, 0);
  }
  int stage = 0;
  for (; row < sh.rows; row += stride, stage ^= 1) {
    const float mean = a.mean[row], rstd = a.rstd[row];
    float u[NS][8], t[NS][8];
    Raw8<T, VEC> rx[NS], rr[NS], rg[NS], ra[NS];
    Kept kept[NS];
    if constexpr (AHEAD) {
      fetch(row + stride, stage ^ 1);
      ring.wait();
#pragma unroll
      for (int s = 0; s < NS; s++) {
        ring.get(stage, 0, s, rx[s]);
        ring.get(stage, 1, s, rg[s]);
        if (a.res) {
          ring.get(stage, slot_res, s, rr[s]);
        }
      }
    } else {
#pragma unroll
      for (int s = 0; s < NS; s++) {
        rx[s].load((const T *)a.x + row * a.x_ld, w0 + s * ws, lane, sh.cols);
        rg[s].load((const T *)a.gy + row * a.gy_ld, w0 + s * ws, lane, sh.cols);
      }
      if (a.res) {
#pragma unroll
        for (int s = 0; s < NS; s++) {
          rr[s].load((const T *)a.res + row * a.res_ld, w0 + s * ws, lane, sh.cols);
        }
      }
      if (a.gh) {
#pragma unroll
        for (int s = 0; s < NS; s++) {
          ra[s].load((const T *)a.gh + row * a.gh_ld, w0 + s * ws, lane, sh.cols);
        }
      }
    }
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int s = 0; s < NS; s++) {
      const int span = w0 + s * sh.warps_per_row;
      float w[8], g[8];
      loadParam<VEC>(a.w, a.w_type, 1.0f, span, lane, sh.cols, w);
      rg[s].get(g);
      if (a.drop) {
        kept[s] = dropped<T, VEC>(key, row, span, lane, sh.cols, rx[s], u[s]);
      } else {
        rx[s].get(u[s]);
        if (a.dx) {
          kept[s] = keepOfSpan<VEC>(key, row, span, lane, sh.cols);
        }
      }
      if (a.res) {
        float r[8];
        rr[s].get(r);
#pragma unroll
        for (int i = 0; i < 8; i++) {
          u[s][i] += r[i];
        }
      }
#pragma unroll
      for (int i = 0; i < 8; i++) {
        // a column past the end has gy = 0 and adds nothing (its u is finite wherever the row's are)
        u[s][i] = (u[s][i] - mean) * rstd;
        dw[s][i] = fmaf(g[i], u[s][i], dw[s][i]);
        db[s][i] += g[i];
        t[s][i] = g[i] * w[i];
        s1 += t[s][i];
        s2 = fmaf(t[s][i], u[s][i], s2);
      }
    }
    const float2 sums = rowSum2<WIDE>(s1, s2, ws, red[stage]);
    // rstd (t - m1 - u m2) + gh
    const float c1 = -sums.x * sh.inv_cols * rstd, c2 = -sums.y * sh.inv_cols * rstd;
#pragma unroll
    for (int s = 0; s < NS; s++) {
      const int span = w0 + s * sh.warps_per_row;
      float d[8];
      if (a.gh) {
        if constexpr (AHEAD) {
          ring.get(stage, slot_gh, s, ra[s]);
        }
        ra[s].get(d);
#pragma unroll
        for (int i = 0; i < 8; i++) {
          d[i] = fmaf(t[s][i], rstd, fmaf(u[s][i], c2, c1)) + d[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
          d[i] = fmaf(t[s][i], rstd, fmaf(u[s][i], c2, c1));
        }
      }
      if (a.dh) {
        storeSpan<T, VEC>((T *)a.dh + row * a.dh_ld, span, lane, sh.cols, d);
      }
      if (a.dx) {
        if constexpr (VEC && sizeof(T) == 2) {
          uint32_t m[4];
          pairMasks(kept[s], m);
#pragma unroll
          for (int i = 0; i < 8; i++) {
            d[i] *= key.scale;
          }
          storeMasked((T *)a.dx + row * a.dx_ld, span, lane, sh.cols, d, m);
        } else {
          dropSpan(key, kept[s], d);
          storeSpan<T, VEC>((T *)a.dx + row * a.dx_ld, span, lane, sh.cols, d);
        }
      }
    }
  }
  if (a.partial == nullptr) {
    return;
  }
  float *out = a.partial + (long long)blockIdx.x * 2 * sh.cols;
  if (!WIDE) {
    // the block's warps have the same columns: they add up one after the other
    float *join = dynamic;
    const int n_warps = blockDim.x >> 5;
    for (int w = 0; w < n_warps; w++) {
      if (warp == w) {
#pragma unroll
        for (int s = 0; s < NS; s++) {
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const int c = Span<VEC>::col(s, lane, i);
            if (c < sh.cols) {
              const float pw = w > 0 ? join[c] : 0.0f, pb = w > 0 ? join[sh.cols + c] : 0.0f;
              (w + 1 < n_warps ? join : out)[c] = pw + dw[s][i];
              (w + 1 < n_warps ? join : out)[sh.cols + c] = pb + db[s][i];
            }
          }
        }
      }
      __syncthreads();
    }
  } else {
#pragma unroll
    for (int s = 0; s < NS; s++) {
      const int span = w0 + s * sh.warps_per_row;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int c = Span<VEC>::col(span, lane, i);
        if (c < sh.cols) {
          out[c] = dw[s][i];
          out[sh.cols + c] = db[s][i];
        }
      }
    }
  }
}

// dw[c] / db[c] = sum over the blocks' partial sums; 32 columns x 32 parts of the blocks per CTA
__global__ void __launch_bounds__(1024)
    normParamKernel(const float *__restrict__ partial, int blocks, int cols, void *dw, void *db, int w_type) {
  pdlEnter();
  __shared__ float part[32][33];
  const int lane = threadIdx.x & 31, q = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane; // over [dw, db]
  float sum = 0.0f;
  if (c < 2 * cols) {
#pragma unroll 4
    for (int b = q; b < blocks; b += 32) {
      sum += partial[(long long)b * 2 * cols + c];
    }
  }
  part[q][lane] = sum;
  __syncthreads();
  sum = warpSum(part[lane][q]);
  const int col = blockIdx.x * 32 + q;
  if (lane == 0 && col < 2 * cols) {
    void *dst = col < cols ? dw : db;
    const int e = col < cols ? col : col - cols;
    if (dst != nullptr) {
      if (w_type == DT_F32) {
        ((float *)dst)[e] = sum;
      } else if (w_type == DT_F16) {
        ((__half *)dst)[e] = __float2half_rn(sum);
      } else {
        ((__nv_bfloat16 *)dst)[e] = __float2bfloat16_rn(sum);
      }
    }
  }
}

// The forward pass gives a warp up to four spans. The backward pass, whose threads hold sums of their columns
// besides, gives it fewer, so that more warps fit: 16384 x 1024 bf16 with dropout took 74 us with four spans to
// a warp and a row to each of eight warps on a multiprocessor, 59 with one span and 32 warps. Above 12
// spans a block of more than 12 warps waits too long at the row's barrier (8192 x 4096 bf16: 108 us with 16 warps, 101
// with eight of two spans, 94 with the next row fetched ahead); above 32 spans (8192 columns) some of
// its registers spill.
NormShape normShape(long long rows, int cols, bool backward) {
  NormShape sh;
  sh.rows = rows;
  sh.cols = cols;
  sh.spans = (cols + 255) / 256;
  sh.per_warp = !backward      ? std::min(sh.spans, 4)
                : sh.spans <= 2  ? sh.spans
                : sh.spans <= 12 ? 1
                : sh.spans <= 32 ? 2
                                 : 4;
  sh.warps_per_row = (sh.spans + sh.per_warp - 1) / sh.per_warp;
  sh.rows_per_block = sh.warps_per_row == 1 ? kRowThreads / 32 : 1;
  sh.inv_cols = 1.0f / (float)cols;
  return sh;
}
int normThreads(const NormShape &sh) { return sh.warps_per_row == 1 ? kRowThreads : sh.warps_per_row * 32; }

// blocks of the backward pass: as many as fit at once, fewer where rows are few
int normGradBlocks(const NormShape &sh) {
  const int warps = normThreads(sh) / 32;
  const long long resident = std::max(1, (sh.warps_per_row > 1 && sh.per_warp == 1 ? 32 : 16) / warps);
  return (int)std::max(1LL, std::min((sh.rows + sh.rows_per_block - 1) / sh.rows_per_block,
                                     resident * digitalSmCount()));
}

template <typename T, bool VEC, bool WIDE, int NS>
void launchForward(const NormShape &sh, const NormFwd &a, const DropKey &key, cudaStream_t stream) {
  const long long blocks = (sh.rows + sh.rows_per_block - 1) / sh.rows_per_block;
  AB200_CUDA(launchChained(normForwardKernel<T, VEC, WIDE, NS>, dim3((unsigned)blocks), dim3(normThreads(sh)), 0, stream,
                           a, sh, key));
  AB200_LAUNCH_CHECK();
}
template <typename T, bool VEC, bool WIDE, int NS>
void launchBackward(const NormShape &sh, const NormBwd &a, const DropKey &key, int blocks, cudaStream_t stream) {
  const size_t smem = normAhead<T>(VEC, WIDE, NS)  ? RowRing<T, NS>::bytes(normTensors(a), normThreads(sh))
                      : a.partial && !WIDE ? (size_t)sh.cols * 2 * sizeof(float)
                                           : 0;
  if (normAhead<T>(VEC, WIDE, NS)) {
    // Always the most that this kernel can ask for (four tensors, 16 warps): the limit counts the kernel's static shared memory
    // as well, and it is state of the kernel, which calls from other threads must not find lowered
    AB200_CUDA(cudaFuncSetAttribute(normBackwardKernel<T, VEC, WIDE, NS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    (int)RowRing<T, NS>::bytes(4, 512)));
  }
  AB200_CUDA(launchChained(normBackwardKernel<T, VEC, WIDE, NS>, dim3((unsigned)blocks), dim3(normThreads(sh)), smem,
                           stream, a, sh, key));
  AB200_LAUNCH_CHECK();
}

template <typename T, bool VEC, typename... Args> void forwardOfShape(const NormShape &sh, Args &&...args) {
  switch (sh.warps_per_row == 1 ? sh.per_warp : 0) {
  case 1: launchForward<T, VEC, false, 1>(sh, args...); break;
  case 2: launchForward<T, VEC, false, 2>(sh, args...); break;
  case 3: launchForward<T, VEC, false, 3>(sh, args...); break;
  case 4: launchForward<T, VEC, false, 4>(sh, args...); break;
  default: launchForward<T, VEC, true, 4>(sh, args...);
  }
}
template <typename T, bool VEC, typename... Args> void backwardOfShape(const NormShape &sh, Args &&...args) {
  if (sh.spans == 1) {
    launchBackward<T, VEC, false, 1>(sh, args...);
  } else if (sh.spans == 2) {
    launchBackward<T, VEC, false, 2>(sh, args...);
  } else if (sh.per_warp == 1) {
    launchBackward<T, VEC, true, 1>(sh, args...);
  } else if (sh.per_warp == 2) {
    launchBackward<T, VEC, true, 2>(sh, args...);
  } else {
    launchBackward<T, VEC, true, 4>(sh, args...);
  }
}

} // namespace

void normForward(const NormArgs &a, cudaStream_t stream) {
  if (a.rows <= 0) {
    return;
  }
  const NormShape sh = normShape(a.rows, a.cols, false);
  const bool vec = a.cols % 8 == 0 && spansAlign(a.x.p, a.x.ld, a.type) &&
                   spansAlign(a.residual.p, a.residual.ld, a.type) && spansAlign(a.y.p, a.y.ld, a.type) &&
                   spansAlign(a.h.p, a.h.ld, a.type) && spansAlign(a.weight, 0, a.w_type) &&
                   spansAlign(a.bias, 0, a.w_type);
  NormFwd k = {a.x.p,     a.residual.p,  a.weight, a.bias,  a.y.p,    a.h.p, a.mean, a.rstd, a.x.ld,
               a.residual.ld, a.y.ld, a.h.ld,   a.w_type, a.eps, a.drop.p > 0.0};
  const DropKey key = dropKey(a.drop);
  switch (a.type) {
  case DT_F32:
    vec ? forwardOfShape<float, true>(sh, k, key, stream) : forwardOfShape<float, false>(sh, k, key, stream);
    break;
  case DT_F16:
    vec ? forwardOfShape<__half, true>(sh, k, key, stream) : forwardOfShape<__half, false>(sh, k, key, stream);
    break;
  default:
    vec ? forwardOfShape<__nv_bfloat16, true>(sh, k, key, stream)
        : forwardOfShape<__nv_bfloat16, false>(sh, k, key, stream);
  }
}

long long normGradWorkspace(long long rows, int cols) {
  return rows <= 0 ? 0 : (long long)normGradBlocks(normShape(rows, cols, true)) * 2 * cols;
}

void normBackward(const NormGradArgs &a, cudaStream_t stream) {
  const NormShape sh = normShape(a.rows, a.cols, true);
  const int blocks = a.rows > 0 ? normGradBlocks(sh) : 0;
  if (blocks > 0) {
    const bool vec = a.cols % 8 == 0 && spansAlign(a.gy.p, a.gy.ld, a.type) && spansAlign(a.gh.p, a.gh.ld, a.type) &&
                     spansAlign(a.x.p, a.x.ld, a.type) && spansAlign(a.residual.p, a.residual.ld, a.type) &&
                     spansAlign(a.dh.p, a.dh.ld, a.type) && spansAlign(a.dx.p, a.dx.ld, a.type) &&
                     spansAlign(a.weight, 0, a.w_type);
    NormBwd k = {a.gy.p,    a.gh.p,  a.x.p,   a.residual.p,  a.weight,  a.dh.p,  a.dx.p,   a.mean,
                 a.rstd,    a.partial, a.gy.ld, a.gh.ld, a.x.ld, a.residual.ld, a.dh.ld, a.dx.ld,
                 a.w_type, a.residual.p != nullptr && a.drop.p > 0.0};
    const DropKey key = dropKey(a.drop);
    switch (a.type) {
    case DT_F32:
      vec ? backwardOfShape<float, true>(sh, k, key, blocks, stream)
          : backwardOfShape<float, false>(sh, k, key, blocks, stream);
      break;
    case DT_F16:
      vec ? backwardOfShape<__half, true>(sh, k, key, blocks, stream)
          : backwardOfShape<__half, false>(sh, k, key, blocks, stream);
      break;
    default:
      vec ? backwardOfShape<__nv_bfloat16, true>(sh, k, key, blocks, stream)
          : backwardOfShape<__nv_bfloat16, false>(sh, k, key, blocks, stream);
    }
  }
  if (a.dweight || a.dbias) {
    AB200_CUDA(launchChained(normParamKernel, dim3((unsigned)((2 * a.cols + 31) / 32)), dim3(1024), 0, stream,
                             (const float *)a.partial, blocks, a.cols, a.dweight, a.dbias, a.w_type));
    AB200_LAUNCH_CHECK();
  }
}

} // namespace ab200
