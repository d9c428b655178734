// Dropout from a counter-based generator: y = keep ? x / (1 - p) : 0 (+ residual). No mask is
// stored; the backward pass is the same kernel on the gradient with the same (seed, call).
// Measured: 16384 x 768 fp32 with residual 22 us (6.9 TB/s), 16384 x 4096 bf16 54 us (5.0 TB/s): with 16-bit
// elements the draws, one Philox block for eight, keep the issue slots and the integer pipe two thirds busy. Fewer
// registers for more warps, or the next spans fetched a turn ahead, made it slower (58 us each).
#include "digital.cuh"

#include <algorithm>
#include <type_traits>

namespace ab200 {

int digitalSmCount() {
  static int count[64] = {};
  int dev = 0;
  AB200_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) {
    int n = 0;
    AB200_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
    return n;
  }
  if (count[dev] == 0) {
    AB200_CUDA(cudaDeviceGetAttribute(&count[dev], cudaDevAttrMultiProcessorCount, dev));
  }
  return count[dev];
}

namespace {

// A warp takes one span of 256 elements at a time, two in flight. FLAT: the rows follow each other
// without a gap and their blocks of eight are numbered alike, so they are one row of up to 2^30 elements.
template <typename T, bool VEC, bool RES, bool FLAT>
__global__ void __launch_bounds__(256)
    dropoutKernel(const T *x, long long x_ld, const T *res, long long res_ld, T *y, long long y_ld, long long rows,
                  int cols, DropKey key) {
  using Index = typename std::conditional<FLAT, uint32_t, long long>::type;
  pdlEnter();
  const int lane = threadIdx.x & 31;
  const uint32_t spans = ((uint32_t)cols + 255u) / 256u;
  const Index total = FLAT ? (Index)spans : (Index)(rows * spans);
  const Index warps = (Index)gridDim.x * (blockDim.x / 32);
  for (Index s = (Index)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32; s < total; s += 2 * warps) {
    Raw8<T, VEC> raw[2], add[2];
    long long row[2];
    int span[2];
#pragma unroll
    for (int q = 0; q < 2; q++) {
      const Index t = s + q * warps;
      if (FLAT) {
        row[q] = 0;
        span[q] = (int)min((uint32_t)t, spans); // past the last span nothing is read or written
      } else {
        row[q] = t >= total ? 0 : total <= 0x7fffffffLL ? (uint32_t)t / spans : t / spans;
        span[q] = t < total ? (int)(t - row[q] * spans) : (int)spans;
      }
      raw[q].load(x + row[q] * x_ld, span[q], lane, cols);
      if (RES) {
        add[q].load(res + row[q] * res_ld, span[q], lane, cols);
      }
    }
#pragma unroll
    for (int q = 0; q < 2; q++) {
      float v[8];
      const Kept kept = keepOfSpan<VEC>(key, row[q], span[q], lane, cols);
      raw[q].get(v);
      if constexpr (VEC && !RES && sizeof(T) == 2) {
        uint32_t m[4];
        pairMasks(kept, m);
#pragma unroll
        for (int i = 0; i < 8; i++) {
          v[i] *= key.scale;
        }
        storeMasked(y + row[q] * y_ld, span[q], lane, cols, v, m);
      } else {
        dropSpan(key, kept, v);
        if (RES) {
          float r[8];
          add[q].get(r);
#pragma unroll
          for (int i = 0; i < 8; i++) {
            v[i] += r[i];
          }
        }
        storeSpan<T, VEC>(y + row[q] * y_ld, span[q], lane, cols, v);
      }
    }
  }
}

template <typename T, bool VEC, bool RES, bool FLAT>
void launchDropout(RowsIn x, RowsIn residual, RowsOut y, long long rows, int cols, const DropKey &key,
                   cudaStream_t stream) {
  const long long total = rows * (((long long)cols + 255) / 256);
  const long long want = (total + 15) / 16;
  const dim3 grid((unsigned)std::max(1LL, std::min(want, (long long)digitalSmCount() * 32)));
  AB200_CUDA(launchChained(dropoutKernel<T, VEC, RES, FLAT>, grid, dim3(256), 0, stream, (const T *)x.p, x.ld,
                           (const T *)residual.p, residual.ld, (T *)y.p, y.ld, rows, cols, key));
  AB200_LAUNCH_CHECK();
}
template <typename T>
void dropoutOfType(RowsIn x, RowsIn residual, RowsOut y, long long rows, int cols, int type, const DropKey &key,
                   cudaStream_t stream) {
  const bool vec = cols % 8 == 0 && spansAlign(x.p, x.ld, type) && spansAlign(y.p, y.ld, type) &&
                   spansAlign(residual.p, residual.ld, type);
  if (!vec) {
    residual.p ? launchDropout<T, false, true, false>(x, residual, y, rows, cols, key, stream)
               : launchDropout<T, false, false, false>(x, residual, y, rows, cols, key, stream);
  } else if (rows == 1 || (x.ld == cols && y.ld == cols && (!residual.p || residual.ld == cols) &&
                           rows * cols <= 0x40000000LL)) {
    cols = (int)(rows * cols);
    residual.p ? launchDropout<T, true, true, true>(x, residual, y, 1, cols, key, stream)
               : launchDropout<T, true, false, true>(x, residual, y, 1, cols, key, stream);
  } else {
    residual.p ? launchDropout<T, true, true, false>(x, residual, y, rows, cols, key, stream)
               : launchDropout<T, true, false, false>(x, residual, y, rows, cols, key, stream);
  }
}

} // namespace

void dropoutApply(RowsIn x, RowsIn residual, RowsOut y, long long rows, int cols, int type, const DropoutArgs &drop,
                  cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) {
    return;
  }
  const DropKey key = dropKey(drop);
  switch (type) {
  case DT_F32: dropoutOfType<float>(x, residual, y, rows, cols, type, key, stream); break;
  case DT_F16: dropoutOfType<__half>(x, residual, y, rows, cols, type, key, stream); break;
  default: dropoutOfType<__nv_bfloat16>(x, residual, y, rows, cols, type, key, stream);
  }
}

} // namespace ab200
