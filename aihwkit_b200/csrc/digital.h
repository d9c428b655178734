// Host entry points of the digital operators around the analog tiles (layer norm, dropout, low-rank
// adapters); the C boundary in capi.cu calls them. Pointers are device memory of the current device.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace ab200 {

enum DigitalType : int { DT_F32 = 0, DT_F16 = 1, DT_BF16 = 2 };

// elements between the starts of two rows; the elements of a row are neighbours
struct RowsIn {
  const void *p;
  long long ld;
};
struct RowsOut {
  void *p;
  long long ld;
};

struct DropoutArgs {
  double p;
  uint64_t seed;
  uint32_t call;
};

struct NormArgs {
  RowsIn x, residual;         // residual.p may be null
  RowsOut y, h;               // h.p may be null
  const void *weight, *bias;  // [cols] or null, of type w_type
  float *mean, *rstd;         // [rows] or null
  long long rows;
  int cols, type, w_type;
  float eps;
  DropoutArgs drop;
};
void normForward(const NormArgs &a, cudaStream_t stream);

struct NormGradArgs {
  RowsIn gy, gh;              // gh.p may be null
  RowsIn x, residual;         // residual.p null: x is h
  RowsOut dh, dx;             // dx.p may be null: then nothing was dropped or dx is not wanted
  const void *weight;         // [cols] or null, of type w_type
  const float *mean, *rstd;   // [rows]
  void *dweight, *dbias;      // [cols] of type w_type, each may be null
  float *partial;             // workspace of normGradWorkspace floats, null when neither is wanted
  long long rows;
  int cols, type, w_type;
  DropoutArgs drop;
};
long long normGradWorkspace(long long rows, int cols);
void normBackward(const NormGradArgs &a, cudaStream_t stream);

void dropoutApply(RowsIn x, RowsIn residual, RowsOut y, long long rows, int cols, int type,
                  const DropoutArgs &drop, cudaStream_t stream);

// Rows of x [rows, k] in segments; segment j has the rows [starts[j], starts[j + 1]) and adapter
// ids[j] (outside [0, adapters): none). starts null: segment j is row j.
struct LowRankRows {
  const int *starts, *ids;
  int segments;
  long long rows;
};
struct LowRankArgs {
  LowRankRows seg;
  RowsIn x, base;             // base.p null: nothing is added
  RowsOut y;                  // y.p null: only v is wanted
  const void *a, *b;          // [adapters, rank, k], [adapters, rank, n]
  const float *scale;         // [adapters]
  float *v;                   // [rows, rank] or null: scale * x a^T
  int k, n, rank, adapters, type;
};
void lowRankApply(const LowRankArgs &a, cudaStream_t stream);

struct LowRankGradArgs {
  LowRankRows seg;
  RowsIn x[2];                // the rows that meet u[0] and u[1]
  const float *u[2];          // [rows, rank]
  void *grad[2];              // [adapters, rank, width], null: not wanted
  int width[2];
  void *workspace;            // lowRankGradWorkspace bytes
  int rank, adapters, type;
};
// width 0: that gradient is not wanted
long long lowRankGradWorkspace(long long rows, int segments, bool one_row_each, int width0, int width1, int rank);
void lowRankGrad(const LowRankGradArgs &a, cudaStream_t stream);

constexpr int kNormMaxCols = 16384;
constexpr int kLowRankMax = 256;

} // namespace ab200
