// Dropout from a counter-based generator: y = keep ? x / (1 - p) : 0 (+ residual). No mask is
// stored; the backward pass is the same kernel on the gradient with the same (seed, call).
#include "digital.cuh"

#include <algorithm>

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

// A warp takes one span of 256 elements at a time, two in flight.
template <typename T, bool VEC, bool RES>
__global__ void __launch_bounds__(256)
    dropoutKernel(const T *x, long long x_ld, const T *res, long long res_ld,
                  T *y, long long y_ld, long long rows, int cols, DropKey key) {
  pdlEnter();
  const int lane = threadIdx.x & 31;
  const int spans = (cols + 255) / 256;
  const long long total = rows * spans;
  const long long warps = (long long)gridDim.x * (blockDim.x / 32);
  for (long long s = (long long)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32; s < total; s += 2 * warps) {
    Raw8<T, VEC> raw[2], add[2];
    long long row[2];
    int span[2];
#pragma unroll
    for (int q = 0; q < 2; q++) {
      const long long t = s + q * warps;
      // past the last span: behind the end of row 0, where nothing is read or written
      row[q] = rows == 1 || t >= total ? 0 : total <= 0x7fffffffLL ? (uint32_t)t / (uint32_t)spans : t / spans;
      span[q] = t < total ? (int)(t - row[q] * spans) : spans;
      raw[q].load(x + row[q] * x_ld, span[q], lane, cols);
      if (RES) {
        add[q].load(res + row[q] * res_ld, span[q], lane, cols);
      }
    }
#pragma unroll
    for (int q = 0; q < 2; q++) {
      float v[8], r[8];
      const uint32_t keep = keepOfSpan<VEC>(key, row[q], span[q], lane, cols);
      raw[q].get(v);
      if (RES) {
        add[q].get(r);
      }
#pragma unroll
      for (int i = 0; i < 8; i++) {
        // a dropped element is zero whatever it held, infinities and NaN included
        v[i] = (keep >> i) & 1u ? v[i] * key.scale : 0.0f;
        if (RES) {
          v[i] += r[i];
        }
      }
      storeSpan<T, VEC>(y + row[q] * y_ld, span[q], lane, cols, v);
    }
  }
}

template <typename T, bool VEC>
void launchDropout(RowsIn x, RowsIn residual, RowsOut y, long long rows, int cols, const DropKey &key,
                   cudaStream_t stream) {
  const long long total = rows * ((cols + 255) / 256);
  const long long want = (total + 15) / 16;
  const dim3 grid((unsigned)std::max(1LL, std::min(want, (long long)digitalSmCount() * 32)));
  if (residual.p) {
    AB200_CUDA(launchChained(dropoutKernel<T, VEC, true>, grid, dim3(256), 0, stream, (const T *)x.p, x.ld,
                             (const T *)residual.p, residual.ld, (T *)y.p, y.ld, rows, cols, key));
  } else {
    AB200_CUDA(launchChained(dropoutKernel<T, VEC, false>, grid, dim3(256), 0, stream, (const T *)x.p, x.ld,
                             (const T *)nullptr, 0LL, (T *)y.p, y.ld, rows, cols, key));
  }
  AB200_LAUNCH_CHECK();
}

} // namespace

void dropoutApply(RowsIn x, RowsIn residual, RowsOut y, long long rows, int cols, int type,
                  const DropoutArgs &drop, cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) {
    return;
  }
  const DropKey key = dropKey(drop);
  bool vec = cols % 8 == 0 && spansAlign(x.p, x.ld, type) && spansAlign(y.p, y.ld, type) &&
             spansAlign(residual.p, residual.ld, type);
  // rows that follow each other without a gap are one row: the blocks of eight are numbered alike
  if (vec && x.ld == cols && y.ld == cols && (!residual.p || residual.ld == cols) &&
      rows * cols <= 0x40000000LL) {
    cols = (int)(rows * cols);
    rows = 1;
  }
  switch (type) {
  case DT_F32:
    vec ? launchDropout<float, true>(x, residual, y, rows, cols, key, stream)
        : launchDropout<float, false>(x, residual, y, rows, cols, key, stream);
    break;
  case DT_F16:
    vec ? launchDropout<__half, true>(x, residual, y, rows, cols, key, stream)
        : launchDropout<__half, false>(x, residual, y, rows, cols, key, stream);
    break;
  default:
    vec ? launchDropout<__nv_bfloat16, true>(x, residual, y, rows, cols, key, stream)
        : launchDropout<__nv_bfloat16, false>(x, residual, y, rows, cols, key, stream);
  }
}

} // namespace ab200
