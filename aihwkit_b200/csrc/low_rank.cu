// Low-rank adapters of many requests beside a shared projection: the rows of request j get
//   y = base + v b[id_j],   v = scale[id_j] x a[id_j]^T,   a [adapters, rank, k], b [adapters, rank, n]
// and the gradients of a and b. With both factors stored rank first, the gradient of x,
// (scale gy b^T) a, is the same operator with the factors' places changed, and the gradients of a
// and b are the same sum over rows, u^T x.
//
// lowRankApplyKernel. The work is narrow: 2 rank operations per element of x and of y, so memory
// bounds it up to ranks of about 64. A block takes up to 64 (32, 16) rows of one request through both
// products: x is read once (above 64 ranks once for every 64), v stays in shared memory, y is written once; nothing but the saved v
// goes through memory between the two. A dot product may run in any order, so a thread takes 16
// neighbouring bytes of a row as its share of k, and columns are dealt to the fragments of mma.sync so that it ends up
// with 16 neighbouring bytes of y. Every warp has its own steps along k and its own columns and
// fetches them with cp.async into a ring of its own, x and a first, then base and b: loads stay in flight through both
// products and the sum between them, and no barrier stands in the loops. Where rows
// are few, a cluster of blocks shares a row tile: each takes a share of k, the partial v are added
// through distributed shared memory in rank order, and each block takes a share of the columns.
// Products: bf16 x bf16 and fp16 x fp16 are exact in the fp32 sum; fp32 factors (v, and x, a, b of
// fp32 calls) are split into two TF32 parts, hi + lo, and multiplied as hi hi + lo hi + hi lo, which leaves
// 2^-22 of a product out. Where v (or u of the gradients) meets bf16, its three parts are bf16 and hold all of its 24
// bits, three products in place of the four that TF32 parts take at half the rate. fp16 has not the range for that.
//
// Measured: 16384 rows 768 -> 2304 rank 16 in 16 requests, fp32 70 us (5.0 TB/s), bf16 38 us (4.6 TB/s); 8192 rows 4096 ->
// 4096 bf16, rank 32 52 us (3.9 TB/s), rank 64 84 us, rank 128 151 us (rank 32 and 64 took 47 and 71 us with v in two bf16 parts);
// 256 tokens of 64 adapters 4096 -> 4096 rank 16 15 us. 16 warps or fewer fit a multiprocessor (registers, rings), and what
// they wait for - loads, shared memory, their own products - bounds it; issue slots are up to 45 % busy, no pipe more than 36 %.
//
// lowRankGradKernel. grad[id] = sum over the rows of id of u^T x: a warp holds rank x 128 bytes of columns
// in fragments and walks a chunk of rows of one request, fetched the same way; chunks' partial sums go
// through memory and are added in the order of the rows (no atomics). Measured: both gradients of 8192 rows 4096 -> 4096
// rank 32 bf16 54 us and 10 us for the chunks' sums (39 and 8 with u in two bf16 parts and one sum of the matrix unit over
// all rows), with 10 warps to a multiprocessor and the matrix pipe half busy.
#include "digital.cuh"

#include <algorithm>
#include <type_traits>

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace ab200 {

namespace {

// These kernels wait for the launch in front of them as the others do, but let the next one start only as they end: blocks
// of a next launch that come early take the places that are free, on few multiprocessors, and stay there.
__device__ __forceinline__ void waitForLaunchBefore() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

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
  int seg;            // the request
  bool alone;         // it has one row
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
    t.alone = true;
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
    t.alone = end == begin + 1;
    seg = lo - 1;
  }
  t.seg = seg;
  t.id = t.rows > 0 && seg >= 0 && seg < s.n ? s.ids[seg] : -1;
  if (t.id >= s.adapters) {
    t.id = -1;
  }
  return t;
}
// Rows of a tile of 16. A request of one row (decoding) shares its tile with the others of one row and the same
// adapter among its 1024 neighbours, sixteen at a time, so that the adapter is read once for them; the first
// of the sixteen keeps the tile, for the others this returns false. All warps of all blocks of a tile find the same.
__device__ __forceinline__ bool gatherRows(const Segments &s, RowTile &tile, int lane, int list[16]) {
  // every place of the list is written by one lane only: ballots order no memory
  if (tile.rows == 1 && tile.id >= 0 && tile.alone) {
    const int first = tile.seg & ~1023, end = min(first + 1024, s.n);
    int before = 0, found = 0; // of the adapter's single rows: ahead of this one, all so far
    for (int w0 = first; w0 < end && found - before < 16; w0 += 256) {
      int id[8], row[8], next[8]; // of 256 requests, all read before the first is looked at
#pragma unroll
      for (int q = 0; q < 8; q++) {
        const int j = w0 + q * 32 + lane;
        id[q] = j < end ? s.ids[j] : -1;
        row[q] = s.starts == nullptr ? j : j < end ? border(s, j + 1) : 0;
        next[q] = s.starts == nullptr ? j + 1 : j < end ? border(s, j + 2) : 0;
      }
#pragma unroll
      for (int q = 0; q < 8; q++) {
        const int w = w0 + q * 32;
        const bool match = id[q] == tile.id && next[q] == row[q] + 1;
        const unsigned hits = __ballot_sync(0xffffffffu, match);
        if (tile.seg >= w) { // up to this row's own place
          before += __popc(tile.seg < w + 32 ? hits & ((1u << (tile.seg - w)) - 1u) : hits);
          if (tile.seg < w + 32 && before % 16 != 0) {
            return false;
          }
        }
        if (tile.seg < w + 32) {
          const int at = found + __popc(hits & ((1u << lane) - 1u)) - before;
          if (match && at >= 0 && at < 16) {
            list[at] = row[q];
          }
        }
        found += __popc(hits);
      }
    }
    tile.rows = min(found - before, 16);
    __syncwarp();
    if (lane >= tile.rows && lane < 16) {
      list[lane] = list[0];
    }
  } else if (lane < 16) {
    list[lane] = tile.row0 + min(lane, tile.rows - 1);
  }
  __syncwarp();
  return true;
}
long long segmentSlots(const LowRankRows &s, int shift) {
  return s.starts ? (s.rows >> shift) + s.segments + 2 : s.rows;
}

// ---- fragments --------------------------------------------------------------------------------
__device__ __forceinline__ void mmaTf32(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},"
               "{%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// the first product of a sum: c = a b
__device__ __forceinline__ void mmaTf32First(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// Four 8 x 16-byte matrices, whose rows are at the addresses of lanes 0-7, 8-15, 16-23 and 24-31: lane l gets word l % 4
// of row l / 4 of each - the operands of mma.sync for 16-bit types and, word by word, for TF32.
__device__ __forceinline__ void loadMatrices(uint32_t src, uint32_t r[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(src)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}
template <typename T>
__device__ __forceinline__ void mma16First(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
  }
}
template <bool SET> __device__ __forceinline__ void setOrAdd(float c[4], const float d[4]) {
#pragma unroll
  for (int e = 0; e < 4; e++) {
    c[e] = SET ? d[e] : c[e] + d[e];
  }
}
// v, or `most` with its sign where it is larger (or NaN: the rest that it is taken from is NaN then)
__device__ __forceinline__ float atMost(float v, float most) {
  float r;
  asm("min.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(most));
  return r;
}
// fp32 = hi + lo, hi the nearest finite value of 11 bits, lo the exact rest (12 bits at most, of which the
// multiplier reads 11; 13 where hi is the largest)
__device__ __forceinline__ void split(float v, uint32_t &hi, uint32_t &lo) {
  hi = __float_as_uint(atMost(__uint_as_float((__float_as_uint(v) + 0x1000u) & 0xffffe000u), __uint_as_float(0x7f7fe000u)));
  lo = __float_as_uint(v - __uint_as_float(hi));
}

// a and b as the halves of a word, in bf16, what is left of them (16 bits at most) in another, and what is left of
// that (8 bits) in a third: fp32 = p[0] + p[1] + p[2]
constexpr int kParts = 3;
constexpr float kMostBf16 = 0x1.fep127f; // fp32 values above would round to infinity
__device__ __forceinline__ void splitPair(float a, float b, uint32_t p[kParts]) {
#pragma unroll
  for (int q = 0; q < kParts; q++) {
    p[q] = q == 0 ? pack2<__nv_bfloat16>(atMost(a, kMostBf16), atMost(b, kMostBf16)) : pack2<__nv_bfloat16>(a, b);
    const float2 f = unpack2<__nv_bfloat16>(p[q]);
    a -= f.x;
    b -= f.y;
  }
}
template <typename T> constexpr bool kPairs = std::is_same<T, __nv_bfloat16>::value;
// bytes of an element of v as an operand of the second product, and the ranks that a product takes (of the gradients: u, rows)
template <typename T> constexpr int kOperandBytes = kPairs<T> ? 2 * kParts : 8;
template <typename T> constexpr int kOperandRanks = kPairs<T> ? 16 : 8;
__host__ __device__ __forceinline__ int operandRanks(int rank) { return (rank + 15) & ~15; }

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

// The matrix unit cuts off what an addition shifts out of its sum, up to 2^-22 of it and always toward zero: with one sum
// going through all products of a row of 16384 positive terms that was 5e-6 of the result, in one direction (65536: 2e-5). So
// it adds up few products at a time (a step's 32 elements of 16-bit types, its 16 of fp32 in three terms; 16 ranks, or 16 to
// 32 rows of the gradients, the smaller parts first), and those sums are added by additions that round.
//
// acc[i][j] += x_i f_j for a step of 64 bytes along k, whose halves h have the operands x[i][h][0..3] and
// f[j][2 h], f[j][2 h + 1]. Each term goes through some fragments before the next: products into one sum
// wait for each other.
template <typename T, int MT, int NT>
__device__ __forceinline__ void mmaStep(float (&acc)[MT][NT][4], uint32_t (&x)[MT][2][4], const uint32_t (&f)[NT][4]) {
  if constexpr (sizeof(T) == 4) {
    // both halves in one sum where the registers hold the sums of all fragments
    constexpr bool BOTH = MT * NT <= 8;
    constexpr int G = BOTH ? NT : 2;
    float sum[MT][G][4];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      uint32_t xl[MT][4];
#pragma unroll
      for (int i = 0; i < MT; i++) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          split(__uint_as_float(x[i][h][e]), x[i][h][e], xl[i][e]);
        }
      }
#pragma unroll
      for (int j0 = 0; j0 < NT; j0 += G) {
        uint32_t fh[G][2], fl[G][2];
#pragma unroll
        for (int j = 0; j < G; j++) {
          split(__uint_as_float(f[j0 + j][2 * h]), fh[j][0], fl[j][0]);
          split(__uint_as_float(f[j0 + j][2 * h + 1]), fh[j][1], fl[j][1]);
        }
#pragma unroll
        for (int term = 0; term < 3; term++) {
#pragma unroll
          for (int j = 0; j < G; j++) {
#pragma unroll
            for (int i = 0; i < MT; i++) {
              if (term == 0 && (h == 0 || !BOTH)) {
                mmaTf32First(sum[i][j], xl[i], fh[j][0], fh[j][1]);
              } else {
                mmaTf32(sum[i][j], term == 0 ? xl[i] : x[i][h], term == 1 ? fl[j][0] : fh[j][0], term == 1 ? fl[j][1] : fh[j][1]);
              }
            }
          }
        }
        if (h == 1 || !BOTH) {
#pragma unroll
          for (int j = 0; j < G; j++) {
#pragma unroll
            for (int i = 0; i < MT; i++) {
              setOrAdd<false>(acc[i][j0 + j], sum[i][j]);
            }
          }
        }
      }
    }
  } else {
    constexpr int G = MT * NT <= 4 ? NT : MT >= 4 ? 1 : 4 / MT; // columns' fragments at a time
#pragma unroll
    for (int j0 = 0; j0 < NT; j0 += G) {
      float sum[MT][G][4];
#pragma unroll
      for (int h = 0; h < 2; h++) {
#pragma unroll
        for (int j = 0; j < G; j++) {
#pragma unroll
          for (int i = 0; i < MT; i++) {
            if (h == 0) {
              mma16First<T>(sum[i][j], x[i][0], f[j0 + j][0], f[j0 + j][1]);
            } else {
              mma16<T>(sum[i][j], x[i][1], f[j0 + j][2], f[j0 + j][3]);
            }
          }
        }
      }
#pragma unroll
      for (int j = 0; j < G; j++) {
#pragma unroll
        for (int i = 0; i < MT; i++) {
          setOrAdd<false>(acc[i][j0 + j], sum[i][j]);
        }
      }
    }
  }
}
// acc[i][j] += sum over STEPS of v_i b_j for the neighbouring columns j of one thread: b0 from row t of a step's eight rows
// of the factor, b1 from row t + 4; partsOf(step, i, parts) gives the upper and the lower part of v_i. FIRST: acc is set, not
// added to
template <typename T, bool FIRST, int STEPS, int MT, int NJ, typename PartsOf>
__device__ __forceinline__ void mmaColumns(float (&acc)[MT][NJ][4], PartsOf partsOf, const uint4 (&b0)[STEPS],
                                           const uint4 (&b1)[STEPS]) {
  uint32_t b[STEPS][NJ][2], bl[STEPS][NJ][2];
#pragma unroll
  for (int step = 0; step < STEPS; step++) {
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      const float f0 = elemOf<T>(b0[step], j), f1 = elemOf<T>(b1[step], j);
      if constexpr (sizeof(T) == 4) {
        split(f0, b[step][j][0], bl[step][j][0]);
        split(f1, b[step][j][1], bl[step][j][1]);
      } else {
        b[step][j][0] = __float_as_uint(f0);
        b[step][j][1] = __float_as_uint(f1);
      }
    }
  }
  constexpr int GJ = NJ < 4 ? NJ : 4, GI = MT < 4 / GJ ? MT : 4 / GJ; // fragments at a time
#pragma unroll
  for (int i0 = 0; i0 < MT; i0 += GI) {
    uint32_t parts[STEPS][GI][2][4];
#pragma unroll
    for (int step = 0; step < STEPS; step++) {
#pragma unroll
      for (int i = 0; i < GI; i++) {
        partsOf(step, i0 + i, parts[step][i]);
      }
    }
#pragma unroll
    for (int j0 = 0; j0 < NJ; j0 += GJ) {
      float sum[GI][GJ][4];
#pragma unroll
      for (int term = 0; term < 3; term++) {
        if (term == 1 && sizeof(T) != 4) {
          continue; // 16-bit factors have no lower part
        }
#pragma unroll
        for (int step = 0; step < STEPS; step++) {
#pragma unroll
          for (int j = 0; j < GJ; j++) {
#pragma unroll
            for (int i = 0; i < GI; i++) {
              const uint32_t (&left)[4] = parts[step][i][term == 0 ? 1 : 0];
              const uint32_t (&right)[2] = term == 1 ? bl[step][j0 + j] : b[step][j0 + j];
              if (term == 0 && step == 0) {
                mmaTf32First(sum[i][j], left, right[0], right[1]);
              } else {
                mmaTf32(sum[i][j], left, right[0], right[1]);
              }
            }
          }
        }
      }
#pragma unroll
      for (int j = 0; j < GJ; j++) {
#pragma unroll
        for (int i = 0; i < GI; i++) {
          setOrAdd<FIRST>(acc[i0 + i][j0 + j], sum[i][j]);
        }
      }
    }
  }
}

// The same for bf16 and sixteen rows of the factor: rows t and t + 4 (b[0], b[1]) go as a pair, and rows t + 8 and
// t + 12 (b[2], b[3]); the parts of their factors come in the same pairs
template <int NJ> __device__ __forceinline__ void pairColumns(const uint4 (&b)[4], uint32_t (&p)[NJ][2]) {
#pragma unroll
  for (int j = 0; j < NJ; j++) {
    const int w = j >> 1;
    const uint32_t pick = (j & 1) ? 0x7632 : 0x5410; // high or low halves of two words
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const uint4 &x = b[2 * h], &y = b[2 * h + 1];
      p[j][h] = __byte_perm(w == 0 ? x.x : w == 1 ? x.y : w == 2 ? x.z : x.w, w == 0 ? y.x : w == 1 ? y.y : w == 2 ? y.z : y.w, pick);
    }
  }
}
template <bool FIRST, int STEPS, int NJ>
__device__ __forceinline__ void mmaPairs(float (&acc)[NJ][4], const uint32_t (&parts)[STEPS][kParts][4],
                                         const uint32_t (&p)[STEPS][NJ][2]) {
#pragma unroll
  for (int j0 = 0; j0 < NJ; j0 += 4) {
    float sum[4][4];
#pragma unroll
    for (int part = kParts - 1; part >= 0; part--) {
#pragma unroll
      for (int step = 0; step < STEPS; step++) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          if (part == kParts - 1 && step == 0) {
            mma16First<__nv_bfloat16>(sum[j], parts[step][part], p[step][j0 + j][0], p[step][j0 + j][1]);
          } else {
            mma16<__nv_bfloat16>(sum[j], parts[step][part], p[step][j0 + j][0], p[step][j0 + j][1]);
          }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
      setOrAdd<FIRST>(acc[j0 + j], sum[j]);
    }
  }
}

// ---- rings of cp.async ------------------------------------------------------------------------
// 16 bytes of a row to shared memory, from `src`, the place of column `col`; columns past the end, and all
// of them where `in` is false, become zeros without a read (nor a branch)
template <typename T>
__device__ __forceinline__ void fetch16B(uint32_t dst, const T *src, int col, int cols, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in && col < cols ? 16 : 0)
               : "memory");
}
// N such pieces, of rows `step` elements apart and STRIDE bytes apart in shared memory, of which the first
// `rows` are there in steps of EVERY from row `first`
template <typename T, int N, int STRIDE, int EVERY>
__device__ __forceinline__ void fetchRows(uint32_t dst, const T *src, long long step, int col, int cols, int first, int rows) {
#pragma unroll
  for (int q = 0; q < N; q++, src += step) {
    fetch16B(dst + q * STRIDE, src, col, cols, q * EVERY + first < rows);
  }
}
// Rows that 16-byte accesses do not fit: N rows of PIECES pieces of 16 bytes from column c0 on, element by element
// with neighbouring lanes on neighbouring elements (a lane that went for its own 16 bytes touched 32 sectors with
// every load: 8192 rows of 2001 -> 2047 rank 16 bf16 took 116 us). fp32 goes by cp.async; 16-bit elements, below what
// it copies, through registers. rowOf gives a row's first element (the next row's is `step` further unless the rows
// come from a LIST), place(row, piece) where a piece goes among its row's.
template <typename T, int N, int PIECES, bool LIST, typename RowOf, typename Place>
__device__ __forceinline__ void fetchOdd(unsigned char *dst, int lane, int c0, int cols, int rows, RowOf rowOf, long long step,
                                         Place place) {
  constexpr int E = 16 / sizeof(T), PER_ROW = PIECES * E; // elements of a row
  constexpr int ROWS = PER_ROW >= 32 ? 1 : 32 / PER_ROW, PARTS = PER_ROW >= 32 ? PER_ROW / 32 : 1;
  const int r0 = lane / (32 / ROWS), e0 = lane % (32 / ROWS);
  const T *next = rowOf(r0) + c0 + e0;
#pragma unroll
  for (int i = 0; i < N / ROWS; i++) {
    const int r = i * ROWS + r0;
    const T *src = LIST ? rowOf(r) + c0 + e0 : next;
#pragma unroll
    for (int h = 0; h < PARTS; h++) {
      const int e = h * 32 + e0;
      const bool in = r < rows && c0 + e < cols;
      unsigned char *at = dst + r * PIECES * 16 + place(r, e / E) * 16 + e % E * (int)sizeof(T);
      if constexpr (sizeof(T) == 4) {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(at)),
                     "l"(src + h * 32), "r"(in ? 4 : 0)
                     : "memory");
      } else {
        *reinterpret_cast<uint16_t *>(at) = in ? reinterpret_cast<const uint16_t *>(src)[h * 32] : (uint16_t)0;
      }
    }
    next += ROWS * step;
  }
}
__device__ __forceinline__ void fetchCommit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// all but the newest N groups of this thread have arrived
template <int N> __device__ __forceinline__ void fetchWait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 shared16B(const unsigned char *src) { return *reinterpret_cast<const uint4 *>(src); }
__device__ __forceinline__ uint4 shared8B(const unsigned char *src) {
  const uint2 q = *reinterpret_cast<const uint2 *>(src);
  return make_uint4(q.x, q.y, 0, 0);
}
template <typename T, bool VEC>
__device__ __forceinline__ void store16B(T *row, int col, int cols, const float *v) {
  constexpr int E = 16 / sizeof(T);
  if (VEC) {
    if (col < cols) {
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(row + col) = make_float4(v[0], v[1], v[2], v[3]);
      } else {
        uint4 q;
        q.x = pack2<T>(v[0], v[1]);
        q.y = pack2<T>(v[2], v[3]);
        q.z = pack2<T>(v[4 % E], v[5 % E]);
        q.w = pack2<T>(v[6 % E], v[7 % E]);
        *reinterpret_cast<uint4 *>(row + col) = q;
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

// MT fragments of 16 rows; ranks go through the products 8 * NT at a time. A stage of a warp's ring has 64
// bytes of each row of x (base) and of 8 * NT rows of a (b). Tiles of 16 rows have eight warps, as
// their time is that of a chain of loads and sums, and the others four.
template <int MT, int NT> struct ApplyShape {
  static constexpr int TM = 16 * MT, RC = 8 * NT, W = MT == 1 ? 8 : 4;
  static constexpr int XB = TM * 64, STAGE = XB + RC * 64;
  static constexpr int STAGES = MT > 1 ? 2 : NT == 4 || NT == 8 ? 3 : 4;
  static constexpr int RING = W * STAGES * STAGE;
  // shares of the warps of a tile of 16 rows, added after one barrier; larger tiles add them in turn
  static constexpr int SHARES = MT == 1 ? W * TM * (RC + 4) * 4 : 0;
  // blocks to a multiprocessor, bounded by registers and shared memory
  static constexpr int BLOCKS = MT == 1 ? 2 : 4;
  template <typename T> static size_t bytes(int rank) {
    const int vs = ((rank + 7) & ~7) + 4;
    return RING + SHARES + (size_t)TM * (operandRanks(rank) * kOperandBytes<T> + vs * 4);
  }
};

template <typename T, bool VEC, int MT, int NT>
__global__ void __launch_bounds__(ApplyShape<MT, NT>::W * 32, (ApplyShape<MT, NT>::BLOCKS)) lowRankApplyKernel(Apply p) {
  using Shape = ApplyShape<MT, NT>;
  constexpr int W = Shape::W, TM = Shape::TM, RC = Shape::RC, S = Shape::STAGES;
  constexpr int E = 16 / sizeof(T), KS = 4 * E; // elements in 16 bytes, of k in a step, of columns in a unit
  constexpr int NJ = E / 2;                     // fragments beside each other in a unit
  extern __shared__ __align__(16) unsigned char smem[];
  waitForLaunchBefore();
  const int part = p.cluster > 1 ? blockIdx.x % p.cluster : 0;
  RowTile tile = findTile(p.seg, blockIdx.x / p.cluster);
  if (tile.rows <= 0) {
    return; // the whole cluster has the same tile
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  __shared__ int tile_rows[MT == 1 ? W : 1][16]; // rows of a tile of 16, a copy for each warp
  if (MT == 1) {
    if (!gatherRows(p.seg, tile, lane, tile_rows[warp])) {
      return; // another tile has this row
    }
  }
  const int units = (p.n + KS - 1) / KS, units_per = (units + p.cluster - 1) / p.cluster;
  const int u_begin_all = min(units, part * units_per), u_end = min(units, part * units_per + units_per);
  const int u_begin = u_begin_all + warp;
  const T *x = (const T *)p.x + tile.row0 * p.x_ld;
  const T *base = (const T *)p.base + tile.row0 * p.base_ld;
  T *y = (T *)p.y + tile.row0 * p.y_ld;
  // rows g and g + 8 of a tile of 16 against row0, and the distance between them; in a larger one they
  // follow each other
  const long long row_g = MT == 1 ? tile_rows[warp][g] - tile.row0 : g;
  const long long row_8 = MT == 1 ? tile_rows[warp][g + 8] - tile_rows[warp][g] : 8;
  if (tile.id < 0) {
    // no adapter: y is base (nothing to do where they are the same memory) or zero
    if (p.y == nullptr || p.y == p.base) {
      return;
    }
    // eight rows of a warp's 512 bytes at a time, all read before the first is written: a block's copy is a
    // chain of such turns, and with fewer rows to a turn it outlasted the tiles that compute
    const int chunks = (u_end - u_begin_all + 7) / 8; // of 512 bytes
    for (int i = warp; i < chunks * ((tile.rows + 7) / 8); i += W) {
      const int col = (u_begin_all + i % chunks * 8) * KS + lane * E, r = i / chunks * 8;
      const bool in = col < u_end * KS;
      uint4 q[8];
#pragma unroll
      for (int j = 0; j < 8; j++) {
        q[j] = p.base && in && r + j < tile.rows ? load16B<T, VEC>(base + (r + j) * p.base_ld, col, p.n) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int j = 0; j < 8; j++) {
        float o[E];
#pragma unroll
        for (int e = 0; e < E; e++) {
          o[e] = elemOf<T>(q[j], e);
        }
        if (in && r + j < tile.rows) {
          store16B<T, VEC>(y + (r + j) * p.y_ld, col, p.n, o);
        }
      }
    }
    return;
  }
  const int r_pad = (p.rank + 7) & ~7, vs = r_pad + 4;
  unsigned char *held = smem + warp * S * Shape::STAGE; // this warp's ring
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(held);
  const int c_end = operandRanks(p.rank);
  // v of the tile as the second product's operands: [fragment][8 ranks (bf16: 16)][parts][lane][4]
  float *v = reinterpret_cast<float *>(smem + Shape::RING);
  float *mine = v + TM * c_end * kOperandBytes<T> / 4; // [TM][vs]: this block's share of v
  float *shares = mine + TM * vs;   // [W][TM][RC + 4], of tiles of 16 rows
  const float scale = p.scale[tile.id];
  const T *fa = (const T *)p.a + (long long)tile.id * p.rank * p.k;
  const T *fb = (const T *)p.b + (long long)tile.id * p.rank * p.n;

  // Addresses are kept as one pointer per operand and advanced: with a product per row and access
  // they were half of all instructions.
  const int rows_in = tile.rows; // rows q * 8 + g below it are there; others are neither fetched nor stored
  const T *x_at = x + row_g * p.x_ld + t * E, *base_at = base + row_g * p.base_ld + t * E;
  T *y_at = y + row_g * p.y_ld + t * E;
  const long long x_8 = row_8 * p.x_ld, base_8 = row_8 * p.base_ld, y_8 = row_8 * p.y_ld;
  const uint32_t own = g * 64 + t * 16; // this thread's 16 bytes of the rows g of a stage
  // While x and a go through, the four 16-byte pieces of a row change places with the row, so that the eight
  // rows of a matrix lie in different banks
  const uint32_t own_x = g * 64 + (t ^ ((g >> 1) & 3)) * 16;
  // and the pieces of b theirs in pairs of rows, for the four rows that a thread's neighbours read with it
  const uint32_t own_b = Shape::XB + g * 64 + (t ^ (g & 2)) * 16;
  const uint32_t read_b = Shape::XB + t * 64 + ((g >> 1) ^ (t & 2)) * 16 + (g & 1) * 8;
  // matrices of x (rows 0-7 and 8-15 of a fragment, two pieces) and of a (eight rows, four pieces)
  const uint32_t mat_row = lane & 15, mat_x = mat_row * 64, mat_swz = (mat_row >> 1) & 3, mat_f = (lane & 7) * 64;

  // row r of the tile against row0, for accesses whose rows are not the thread's own
  const auto rowAt = [&](int r) { return MT == 1 ? (long long)(tile_rows[warp][r] - tile.row0) : (long long)r; };

  // v = x a^T: steps of KS along k are dealt to the blocks of the cluster and to the warps in turn
  const int steps = (p.k + KS - 1) / KS, steps_per = (steps + p.cluster - 1) / p.cluster;
  const int s_begin = part * steps_per + warp, s_end = min(steps, part * steps_per + steps_per);
  // y = base + v b: units of KS columns, and for each RC ranks at a time; base comes with the last ranks
  int f_unit = p.y != nullptr ? u_begin : units, f_rank = 0, f_stage = 0; // what fetchUnit takes next
  const auto fetchUnit = [&]() {
    if (f_unit < u_end) {
      const int c0 = f_unit * KS, col = c0 + t * E;
      const bool last = f_rank + RC >= p.rank;
      const bool with_base = p.base != nullptr && last;
      if constexpr (VEC) {
        const uint32_t dst = ring + f_stage * Shape::STAGE;
        if (with_base) {
          fetchRows<T, 2 * MT, 512, 8>(dst + own, base_at + c0, base_8, col, p.n, g, rows_in);
        }
        fetchRows<T, NT, 512, 8>(dst + own_b, fb + (long long)(f_rank + g) * p.n + col, 8LL * p.n, col, p.n, f_rank + g, p.rank);
      } else {
        unsigned char *dst = held + f_stage * Shape::STAGE;
        if (with_base) {
          fetchOdd<T, TM, 4, MT == 1>(dst, lane, c0, p.n, rows_in, [&](int r) { return base + rowAt(r) * p.base_ld; }, p.base_ld,
                                      [](int, int piece) { return piece; });
        }
        fetchOdd<T, RC, 4, false>(dst + Shape::XB, lane, c0, p.n, p.rank - f_rank,
                                  [&](int r) { return fb + (long long)(f_rank + r) * p.n; }, p.n,
                                  [](int r, int piece) { return piece ^ (r & 2); });
      }
      f_rank = last ? 0 : f_rank + RC;
      f_unit += last ? W : 0;
    }
    f_stage = f_stage + 1 == S ? 0 : f_stage + 1;
    fetchCommit();
  };
  for (int r0 = 0; r0 < p.rank; r0 += RC) {
    float acc[MT][NT][4];
#pragma unroll
    for (int i = 0; i < MT; i++) {
#pragma unroll
      for (int j = 0; j < NT; j++) {
        acc[i][j][0] = acc[i][j][1] = acc[i][j][2] = acc[i][j][3] = 0.0f;
      }
    }
    const auto fetchStep = [&](int s, int stage) {
      if (s < s_end) {
        const int c0 = s * KS, k0 = c0 + t * E;
        if constexpr (VEC) {
          const uint32_t dst = ring + stage * Shape::STAGE + own_x;
          fetchRows<T, 2 * MT, 512, 8>(dst, x_at + c0, x_8, k0, p.k, g, rows_in);
          fetchRows<T, NT, 512, 8>(dst + Shape::XB, fa + (long long)(r0 + g) * p.k + k0, 8LL * p.k, k0, p.k, r0 + g, p.rank);
        } else {
          unsigned char *dst = held + stage * Shape::STAGE;
          const auto swizzled = [](int r, int piece) { return piece ^ ((r >> 1) & 3); };
          fetchOdd<T, TM, 4, MT == 1>(dst, lane, c0, p.k, rows_in, [&](int r) { return x + rowAt(r) * p.x_ld; }, p.x_ld, swizzled);
          fetchOdd<T, RC, 4, false>(dst + Shape::XB, lane, c0, p.k, p.rank - r0,
                                    [&](int r) { return fa + (long long)(r0 + r) * p.k; }, p.k, swizzled);
        }
      }
      fetchCommit();
    };
#pragma unroll
    for (int q = 0; q < S - 1; q++) {
      fetchStep(s_begin + q * W, q);
    }
    int stage = 0;
    for (int s = s_begin; s < s_end; s += W) {
      __syncwarp(); // all lanes have read the stage that is filled now
      fetchStep(s + (S - 1) * W, stage == 0 ? S - 1 : stage - 1);
      fetchWait<S - 1>();
      __syncwarp(); // and see what the others fetched
      const uint32_t src = ring + stage * Shape::STAGE;
      uint32_t xf[MT][2][4], f[NT][4];
#pragma unroll
      for (int i = 0; i < MT; i++) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
          loadMatrices(src + i * 1024 + mat_x + (((2 * h + (lane >> 4)) ^ mat_swz) * 16), xf[i][h]);
        }
      }
#pragma unroll
      for (int j = 0; j < NT; j++) {
        loadMatrices(src + Shape::XB + j * 512 + mat_f + (((lane >> 3) ^ ((lane >> 1) & 3)) * 16), f[j]);
      }
      mmaStep<T>(acc, xf, f);
      stage = stage + 1 == S ? 0 : stage + 1;
    }
    __syncwarp();
    if (r0 + RC >= p.rank) {
      // the ring is read: the first units arrive while the shares of v are added
#pragma unroll
      for (int q = 0; q < S - 1; q++) {
        fetchUnit();
      }
    }
    if (MT == 1) {
#pragma unroll
      for (int j = 0; j < NT; j++) {
        float *d = shares + (warp * TM + g) * (RC + 4) + j * 8 + 2 * t;
        *reinterpret_cast<float2 *>(d) = make_float2(acc[0][j][0], acc[0][j][1]);
        *reinterpret_cast<float2 *>(d + 8 * (RC + 4)) = make_float2(acc[0][j][2], acc[0][j][3]);
      }
      __syncthreads();
      for (int e = threadIdx.x; e < TM * RC; e += W * 32) {
        const int r = e / RC, c = e % RC;
        if (r0 + c < r_pad) {
          float sum = 0.0f;
#pragma unroll
          for (int w = 0; w < W; w++) {
            sum += shares[(w * TM + r) * (RC + 4) + c];
          }
          mine[r * vs + r0 + c] = sum;
        }
      }
      __syncthreads();
      continue;
    }
    // the warps add their shares one after the other
    for (int w = 0; w < W; w++) {
      if (warp == w) {
#pragma unroll
        for (int i = 0; i < MT; i++) {
#pragma unroll
          for (int j = 0; j < NT; j++) {
            if (r0 + j * 8 < r_pad) {
              float2 *d = reinterpret_cast<float2 *>(mine + (i * 16 + g) * vs + r0 + j * 8 + 2 * t);
              float2 *d8 = reinterpret_cast<float2 *>(mine + (i * 16 + g + 8) * vs + r0 + j * 8 + 2 * t);
              float2 c = make_float2(acc[i][j][0], acc[i][j][1]), c8 = make_float2(acc[i][j][2], acc[i][j][3]);
              if (w > 0) {
                const float2 o = *d, o8 = *d8;
                c.x += o.x;
                c.y += o.y;
                c8.x += o8.x;
                c8.y += o8.y;
              }
              *d = c;
              *d8 = c8;
            }
          }
        }
      }
      __syncthreads();
    }
  }
  cg::cluster_group cluster = cg::this_cluster();
  if (p.cluster > 1) {
    cluster.sync();
  }
  for (int r = threadIdx.x / 8; r < TM; r += W * 4) {
    for (int c = threadIdx.x % 8; c < c_end; c += 8) {
      float sum = 0.0f;
      if (c >= r_pad) {
      } else if (p.cluster > 1) {
        float share[8]; // all on their way before the first is added
#pragma unroll
        for (int q = 0; q < 8; q++) {
          share[q] = q < p.cluster ? cluster.map_shared_rank(mine, q)[r * vs + c] : 0.0f;
        }
#pragma unroll
        for (int q = 0; q < 8; q++) {
          sum += share[q];
        }
      } else {
        sum = mine[r * vs + c];
      }
      sum *= scale;
      if constexpr (kPairs<T>) {
        __nv_bfloat16 *d = reinterpret_cast<__nv_bfloat16 *>(v) +
                           (((r / 16 * (c_end / 16) + c / 16) * 32 * kParts + r % 8 * 4 + c % 4) * 4 + (r % 16) / 8 + (c % 16) / 8 * 2) * 2 +
                           (c % 8) / 4;
        float left = sum;
#pragma unroll
        for (int q = 0; q < kParts; q++) {
          const __nv_bfloat16 part = __float2bfloat16_rn(q == 0 ? atMost(left, kMostBf16) : left);
          d[q * 256] = part;
          left -= __bfloat162float(part);
        }
      } else {
        uint32_t hi, lo;
        split(sum, hi, lo);
        float *d = v + ((r / 16 * (c_end / 8) + c / 8) * 64 + r % 8 * 4 + c % 4) * 4 + (r % 16) / 8 + (c % 8) / 4 * 2;
        d[0] = __uint_as_float(hi);
        d[128] = __uint_as_float(lo);
      }
      if (p.v != nullptr && part == 0 && r < tile.rows && c < p.rank) {
        const long long row = MT == 1 ? tile_rows[warp][r] : tile.row0 + r;
        p.v[row * p.rank + c] = sum;
      }
    }
  }
  if (p.cluster > 1) {
    cluster.sync(); // no block leaves before all have read its share
  } else {
    __syncthreads();
  }
  if (p.y == nullptr) {
    return;
  }
  if (VEC && p.base == nullptr) { // zeros in its place, in every stage (each thread reads its own)
    for (int q = 0; q < S * 2 * MT; q++) {
      *reinterpret_cast<uint4 *>(smem + warp * S * Shape::STAGE + q / (2 * MT) * Shape::STAGE + own + q % (2 * MT) * 512) =
          make_uint4(0, 0, 0, 0);
    }
  }
  float acc[MT][NJ][4];
  const uint4 *operands = reinterpret_cast<const uint4 *>(v) + lane;
  int stage = 0, r0 = 0;
  for (int u = u_begin; u < u_end;) {
    __syncwarp(); // all lanes have read the stage that is filled now
    fetchUnit();
    fetchWait<S - 1>();
    __syncwarp(); // b is read by other lanes than fetched it
    unsigned char *held_now = held + stage * Shape::STAGE;
    const unsigned char *src = held_now;
    stage = stage + 1 == S ? 0 : stage + 1;
    constexpr int RS = kOperandRanks<T>, PARTS = kPairs<T> ? kParts : 2;
    constexpr int STEPS = kPairs<T> || NT == 1 ? 1 : 2; // products to a sum
    const auto ranks = [&](int r, auto first) {
      const auto partsOf = [&](int step, int m, uint32_t (&parts)[PARTS][4]) {
#pragma unroll
        for (int part = 0; part < PARTS; part++) {
          const uint4 q = operands[((m * (c_end / RS) + (r0 + r) / RS + step) * PARTS + part) * 32];
          parts[part][0] = q.x, parts[part][1] = q.y, parts[part][2] = q.z, parts[part][3] = q.w;
        }
      };
      if constexpr (kPairs<T>) {
        uint4 b[4];
#pragma unroll
        for (int q = 0; q < 4; q++) {
          b[q] = r + q * 4 < RC ? shared8B(src + read_b + (r + q * 4) * 64) : make_uint4(0, 0, 0, 0);
        }
        uint32_t pairs[1][NJ][2];
        pairColumns(b, pairs[0]);
#pragma unroll
        for (int m = 0; m < MT; m++) {
          uint32_t parts[1][PARTS][4];
          partsOf(0, m, parts[0]);
          mmaPairs<decltype(first)::value, 1>(acc[m], parts, pairs);
        }
      } else {
        uint4 b0[STEPS], b1[STEPS];
#pragma unroll
        for (int step = 0; step < STEPS; step++) {
          b0[step] = shared8B(src + read_b + (r + step * 8) * 64);
          b1[step] = shared8B(src + read_b + (r + step * 8 + 4) * 64);
        }
        mmaColumns<T, decltype(first)::value, STEPS>(acc, partsOf, b0, b1);
      }
    };
    if (NT < 8 || r0 == 0) { // kernels of fewer than 64 ranks have them all in one pass
      ranks(0, std::true_type());
    } else {
      ranks(0, std::false_type());
    }
#pragma unroll
    for (int r = RS * STEPS; r < RC; r += RS * STEPS) {
      if (r0 + r < p.rank) {
        ranks(r, std::false_type());
      }
    }
    if (NT == 8 && r0 + RC < p.rank) {
      r0 += RC;
      continue;
    }
    const int col = u * KS + t * E;
    T *dst = y_at + u * KS;
#pragma unroll
    for (int q = 0; q < 2 * MT; q++, dst += y_8) {
      if (q * 8 + g < rows_in) {
        const uint4 old = VEC || p.base != nullptr ? shared16B(src + own + q * 512) : make_uint4(0, 0, 0, 0);
        float o[E];
#pragma unroll
        for (int j = 0; j < NJ; j++) {
          o[j] = acc[q / 2][j][2 * (q % 2)] + elemOf<T>(old, j);
          o[NJ + j] = acc[q / 2][j][2 * (q % 2) + 1] + elemOf<T>(old, NJ + j);
        }
        if constexpr (VEC) {
          if (col < p.n) {
            store16B<T, true>(dst, 0, E, o);
          }
        } else {
          store16B<T, true>(reinterpret_cast<T *>(held_now + own + q * 512), 0, E, o);
        }
      }
    }
    if constexpr (!VEC) {
      // the unit's results are in base's place: out by rows, neighbouring lanes on neighbouring elements
      __syncwarp();
      constexpr int ROWS = 32 / KS; // rows a turn
      const int e = lane % KS;
#pragma unroll 8
      for (int r = lane / KS; r < rows_in; r += ROWS) {
        if (u * KS + e < p.n) {
          y[rowAt(r) * p.y_ld + u * KS + e] = reinterpret_cast<const T *>(held_now + r * 64)[e];
        }
      }
    }
    r0 = 0;
    u += W;
  }
}

constexpr long long kSharedPerSm = 228 * 1024; // of which each block takes 1 KB besides its own

template <typename T, bool VEC, int MT, int NT>
void launchApply(Apply p, const LowRankRows &seg, int shift, cudaStream_t stream) {
  p.seg.shift = shift;
  const long long slots = segmentSlots(seg, shift);
  // Blocks that share a tile: as many as fit the GPU at once, eight at most. Of tiles of one row, those
  // that find others of their adapter make one; of 256 rows with 64 adapters about 80 stay.
  const long long active = MT == 1 ? std::min(slots, p.seg.adapters + slots / 16) : slots;
  const size_t smem = ApplyShape<MT, NT>::template bytes<T>(p.rank);
  const long long fit = std::min<long long>(ApplyShape<MT, NT>::BLOCKS, kSharedPerSm / (smem + 1024));
  p.cluster = 1;
  while (p.cluster < 8 && active * p.cluster * 2 <= fit * digitalSmCount()) {
    p.cluster *= 2;
  }
  auto kernel = lowRankApplyKernel<T, VEC, MT, NT>;
  // Always the most that this kernel can ask for: the limit is state of the kernel, and a call from another thread must not find
  // it lowered between its own setting and its launch
  constexpr int kMostRanks = NT == 8 ? kLowRankMax : 8 * NT;
  AB200_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  (int)ApplyShape<MT, NT>::template bytes<T>(kMostRanks)));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(slots * p.cluster));
  cfg.blockDim = dim3(ApplyShape<MT, NT>::W * 32);
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
template <typename T, bool VEC> void dispatchApply(const Apply &p, const LowRankRows &seg, cudaStream_t st) {
  // Requests of 16 rows and fewer on average (decoding) take tiles of 16 rows, longer ones of 64, or 32 with
  // more than 16 ranks: with the fragments of 64 rows only three blocks fitted a multiprocessor (8192 rows,
  // 4096 -> 4096, rank 32, bf16: 78 us, 51 with 32 rows). 32 rows, too, where elements are fetched one by
  // one (8192 x 2001 -> 2047 rank 16 fp32: 93 us with 64 rows, 71 with 32)
  constexpr int kLong = VEC ? 4 : 2, kLongShift = kLong == 4 ? 6 : 5;
  if (seg.starts == nullptr || seg.rows <= 16LL * seg.segments) {
    if (p.rank <= 8) {
      launchApply<T, VEC, 1, 1>(p, seg, 4, st);
    } else if (p.rank <= 16) {
      launchApply<T, VEC, 1, 2>(p, seg, 4, st);
    } else if (p.rank <= 32) {
      launchApply<T, VEC, 1, 4>(p, seg, 4, st);
    } else {
      launchApply<T, VEC, 1, 8>(p, seg, 4, st);
    }
  } else if (p.rank <= 8) {
    launchApply<T, VEC, kLong, 1>(p, seg, kLongShift, st);
  } else if (p.rank <= 16) {
    launchApply<T, VEC, kLong, 2>(p, seg, kLongShift, st);
  } else if (p.rank <= 32) {
    launchApply<T, VEC, 2, 4>(p, seg, 5, st);
  } else {
    launchApply<T, VEC, 2, 8>(p, seg, 5, st);
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
  int block0; // first block of columns of this launch
};

constexpr int kGradWarps = 4, kGradRows = 32, kGradStages = 3;

// a stage: 32 rows of 128 bytes for every warp, and the ranks of the same rows of u for all of them (rows of
// 16 RT + 8 floats: the eight ranks x four rows of a fragment then lie in different banks). Behind the ring the parts of
// u of the present stage, as the products' operands, split once for the four warps (both gradients of 8192 rows 4096 -> 4096
// rank 32 bf16: 66 us with a split for each warp, 61 with one; 60 with 32 rows to a sum of the matrix unit)
template <typename T, int RT> struct GradShape {
  static constexpr int US = 16 * RT + 8;
  static constexpr int XB = kGradRows * 128, STAGE = kGradWarps * XB + kGradRows * US * 4;
  static constexpr int RING = kGradStages * STAGE, BYTES = RING + kGradRows * 16 * RT * kOperandBytes<T>;
};

template <typename T, bool VEC, int RT>
__global__ void __launch_bounds__(kGradWarps * 32, RT == 4 ? 2 : 3) lowRankGradKernel(Grad p) {
  using Shape = GradShape<T, RT>;
  constexpr int E = 16 / sizeof(T), NJ = E, UC = 8 * NJ, S = kGradStages;
  constexpr int RS = kOperandRanks<T>, PARTS = kPairs<T> ? kParts : 2; // rows to a product
  extern __shared__ __align__(16) unsigned char smem[];
  waitForLaunchBefore();
  const int side = blockIdx.z / p.rank_passes, r0 = (blockIdx.z % p.rank_passes) * 16 * RT;
  const RowTile tile = findTile(p.seg, blockIdx.x);
  const int column_block = p.block0 + (int)blockIdx.y;
  if (column_block == 0 && blockIdx.z == 0 && threadIdx.x == 0) {
    p.slot_id[blockIdx.x] = tile.rows > 0 ? tile.id : -1;
  }
  const int width = side ? p.width[1] : p.width[0];
  const long long ld = side ? p.x_ld[1] : p.x_ld[0];
  float *partial = side ? p.partial[1] : p.partial[0];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  if (tile.rows <= 0 || tile.id < 0 || partial == nullptr || column_block * kGradWarps * UC >= width) {
    return; // all threads alike
  }
  const int unit = column_block * kGradWarps + warp; // may lie past the width: all its columns are zeros then
  const T *x = (const T *)(side ? p.x[1] : p.x[0]) + tile.row0 * ld;
  const float *u = (side ? p.u[1] : p.u[0]) + (long long)tile.row0 * p.rank + r0;
  const int ranks = min(p.rank - r0, 16 * RT);
  const bool u_wide = p.rank % 4 == 0 && (uintptr_t)u % 16 == 0;
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem);
  uint4 *operands = reinterpret_cast<uint4 *>(smem + Shape::RING);
  const int chunks = (tile.rows + kGradRows - 1) / kGradRows;
  const auto fetch = [&](int i, int stage) {
    if (i < chunks) {
      const uint32_t dst = ring + stage * Shape::STAGE;
      const int row0 = i * kGradRows, rows = tile.rows - row0;
      // pieces change places with the row, so that four rows of a fragment lie in different banks
      if constexpr (VEC) {
        const int col = unit * UC + (lane & 7) * E;
        const uint32_t mine = dst + warp * Shape::XB + (lane >> 3) * 128 + ((lane & 7) ^ (2 * (lane >> 3))) * 16;
        fetchRows<T, kGradRows / 4, 512, 4>(mine, x + (row0 + (lane >> 3)) * ld + col, 4 * ld, col, width, lane >> 3, rows);
      } else {
        fetchOdd<T, kGradRows, 8, false>(smem + stage * Shape::STAGE + warp * Shape::XB, lane, unit * UC, width, rows,
                                         [&](int r) { return x + (row0 + r) * ld; }, ld,
                                         [](int r, int piece) { return piece ^ (2 * (r & 3)); });
      }
      if (u_wide) {
        for (int e = threadIdx.x; e < kGradRows * 4 * RT; e += kGradWarps * 32) {
          const int r = e / (4 * RT), c = e % (4 * RT) * 4;
          fetch16B(dst + kGradWarps * Shape::XB + (r * Shape::US + c) * 4, u + (long long)(row0 + r) * p.rank + c,
                                c, ranks, r < rows);
        }
      } else {
        for (int e = threadIdx.x; e < kGradRows * 16 * RT; e += kGradWarps * 32) {
          const int r = e / (16 * RT), c = e % (16 * RT);
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + kGradWarps * Shape::XB +
                                                                           (r * Shape::US + c) * 4),
                       "l"(u + (long long)(row0 + r) * p.rank + c), "r"(r < rows && c < ranks ? 4 : 0)
                       : "memory");
        }
      }
    }
    fetchCommit();
  };
  float acc[RT][NJ][4];
#pragma unroll
  for (int i = 0; i < RT; i++) {
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      acc[i][j][0] = acc[i][j][1] = acc[i][j][2] = acc[i][j][3] = 0.0f;
    }
  }
#pragma unroll
  for (int q = 0; q < S - 1; q++) {
    fetch(q, q);
  }
  for (int i = 0; i < chunks; i++) {
    fetchWait<S - 2>();
    __syncthreads(); // chunk i is there for all, and all are done with the stage and the operands of chunk i - 1
    fetch(i + S - 1, (i + S - 1) % S);
    const unsigned char *src = smem + (i % S) * Shape::STAGE;
    const float *us = reinterpret_cast<const float *>(src + kGradWarps * Shape::XB);
    const unsigned char *xs = src + warp * Shape::XB + t * 128 + (g ^ (2 * t)) * 16;
    // the parts of u: [step of RS rows][fragment of 16 ranks][part][lane][4]
    for (int item = warp; item < kGradRows / RS * RT; item += kGradWarps) {
      const float *uf = us + (item / RT * RS + t) * Shape::US + item % RT * 16 + g;
      uint32_t parts[PARTS][4];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float *f = uf + (e >> 1) * (RS / 2) * Shape::US + (e & 1) * 8;
        if constexpr (kPairs<T>) {
          uint32_t pair[kParts];
          splitPair(f[0], f[4 * Shape::US], pair);
#pragma unroll
          for (int part = 0; part < kParts; part++) {
            parts[part][e] = pair[part];
          }
        } else {
          split(f[0], parts[0][e], parts[1][e]);
        }
      }
#pragma unroll
      for (int part = 0; part < PARTS; part++) {
        operands[(item * PARTS + part) * 32 + lane] = make_uint4(parts[part][0], parts[part][1], parts[part][2], parts[part][3]);
      }
    }
    __syncthreads();
    constexpr int STEPS = 2; // products to a sum
#pragma unroll 1
    for (int r = 0; r < kGradRows; r += RS * STEPS) {
      const auto partsOf = [&](int step, int q, uint32_t (&parts)[PARTS][4]) {
#pragma unroll
        for (int part = 0; part < PARTS; part++) {
          const uint4 w = operands[(((r / RS + step) * RT + q) * PARTS + part) * 32 + lane];
          parts[part][0] = w.x, parts[part][1] = w.y, parts[part][2] = w.z, parts[part][3] = w.w;
        }
      };
      if constexpr (kPairs<T>) {
        uint32_t pairs[STEPS][NJ][2];
#pragma unroll
        for (int step = 0; step < STEPS; step++) {
          uint4 b[4];
#pragma unroll
          for (int q = 0; q < 4; q++) {
            b[q] = shared16B(xs + (r + step * RS + 4 * q) * 128);
          }
          pairColumns(b, pairs[step]);
        }
#pragma unroll
        for (int q = 0; q < RT; q++) {
          uint32_t parts[STEPS][PARTS][4];
#pragma unroll
          for (int step = 0; step < STEPS; step++) {
            partsOf(step, q, parts[step]);
          }
          mmaPairs<false, STEPS>(acc[q], parts, pairs);
        }
      } else {
        uint4 x0[STEPS], x1[STEPS];
#pragma unroll
        for (int step = 0; step < STEPS; step++) {
          x0[step] = shared16B(xs + (r + step * RS) * 128);
          x1[step] = shared16B(xs + (r + step * RS + 4) * 128);
        }
        mmaColumns<T, false, STEPS>(acc, partsOf, x0, x1);
      }
    }
  }
  const int col = unit * UC + 2 * NJ * t;
  float *out = partial + ((long long)blockIdx.x * p.rank + r0) * width;
#pragma unroll
  for (int i = 0; i < RT; i++) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int r = i * 16 + h * 8 + g;
      float *at = out + (long long)r * width + col;
      if (r < ranks && VEC) {
#pragma unroll
        for (int j = 0; j < 2 * NJ; j += 4) {
          if (col + j < width) {
            *reinterpret_cast<float4 *>(at + j) =
                make_float4(acc[i][j % NJ][2 * h + j / NJ], acc[i][j % NJ + 1][2 * h + j / NJ],
                            acc[i][j % NJ + 2][2 * h + j / NJ], acc[i][j % NJ + 3][2 * h + j / NJ]);
          }
        }
      } else if (r < ranks) {
#pragma unroll
        for (int j = 0; j < 2 * NJ; j++) {
          if (col + j < width) {
            at[j] = acc[i][j % NJ][2 * h + j / NJ];
          }
        }
      }
    }
  }
}

// grad[i] = sum of the partial sums of adapter i's chunks; zero without any. A warp has 32 elements; where
// elements are few, the warps of a block share them (SHARED), warp w taking the adapter's chunks w, w + 8, ... The
// chunks go in the order of the rows, so the order of the sum is fixed.
constexpr int kJoinWarps = 8;
template <typename T, bool SHARED>
__global__ void __launch_bounds__(kJoinWarps * 32)
    lowRankJoinKernel(const int *__restrict__ slot_id, int slots, const float *__restrict__ p0,
                      const float *__restrict__ p1, T *g0, T *g1, long long elems0, long long elems1) {
  waitForLaunchBefore();
  __shared__ float part[kJoinWarps][32];
  const int side = blockIdx.z, i = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long elems = side ? elems1 : elems0;
  const float *partial = side ? p1 : p0;
  T *grad = side ? g1 : g0;
  const long long e = ((long long)blockIdx.x * (SHARED ? 1 : kJoinWarps) + (SHARED ? 0 : warp)) * 32 + lane;
  if (grad == nullptr) {
    return;
  }
  const float *mine = partial + (e < elems ? e : 0);
  float sum = 0.0f;
  int seen = 0; // chunks of the adapter before these 32
  for (int s0 = 0; s0 < slots; s0 += 32) {
    unsigned left = __ballot_sync(0xffffffffu, s0 + lane < slots && slot_id[s0 + lane] == i);
    while (left != 0) {
      float v[4]; // four chunks on their way before the first is added
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const bool take = left != 0 && (!SHARED || seen % kJoinWarps == warp);
        v[q] = take ? mine[(long long)(s0 + __ffs(left) - 1) * elems] : 0.0f;
        seen += left != 0 ? 1 : 0;
        left &= left - 1;
      }
#pragma unroll
      for (int q = 0; q < 4; q++) {
        sum += v[q];
      }
    }
  }
  if (SHARED) {
    part[warp][lane] = sum;
    __syncthreads();
    if (warp != 0) {
      return;
    }
#pragma unroll
    for (int w = 1; w < kJoinWarps; w++) {
      sum += part[w][lane];
    }
  }
  if (e < elems) {
    grad[i * elems + e] = Elem<T>::put(sum);
  }
}

// rows per chunk: enough blocks for two per multiprocessor, between 128 and 2048 rows
int gradShift(const LowRankRows &s, int width0, int width1) {
  int shift = 11;
  const long long units = (width0 + width1 + 255) / 256;
  while (shift > 7 && units * (s.rows >> shift) < 2LL * digitalSmCount()) {
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
  auto kernel = rt == 1 ? lowRankGradKernel<T, VEC, 1> : rt == 2 ? lowRankGradKernel<T, VEC, 2> : lowRankGradKernel<T, VEC, 4>;
  const int smem = rt == 1 ? GradShape<T, 1>::BYTES : rt == 2 ? GradShape<T, 2>::BYTES : GradShape<T, 4>::BYTES;
  AB200_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  // a grid's second dimension takes 65535 blocks: rows of more than 8388480 fp32 columns go in parts
  const int blocks = (widest + uc - 1) / uc;
  for (p.block0 = 0; p.block0 < blocks; p.block0 += 65535) {
    const dim3 grid((unsigned)slots, (unsigned)std::min(blocks - p.block0, 65535), (unsigned)(2 * p.rank_passes));
    AB200_CUDA(launchChained(kernel, grid, dim3(kGradWarps * 32), smem, st, p));
    AB200_LAUNCH_CHECK();
  }
}
template <typename T>
void gradOfType(const Grad &p, const LowRankGradArgs &a, long long slots, bool vec, cudaStream_t st) {
  if (slots > 0) {
    vec ? launchGrad<T, true>(p, slots, st) : launchGrad<T, false>(p, slots, st);
  }
  const long long e0 = (long long)a.rank * a.width[0], e1 = (long long)a.rank * a.width[1];
  const long long most = std::max(a.grad[0] ? e0 : 0, a.grad[1] ? e1 : 0);
  const long long warps = (most + 31) / 32;
  const bool shared = warps * a.adapters < 4LL * digitalSmCount();
  auto join = shared ? lowRankJoinKernel<T, true> : lowRankJoinKernel<T, false>;
  AB200_CUDA(launchChained(join, dim3((unsigned)(shared ? warps : (warps + kJoinWarps - 1) / kJoinWarps), (unsigned)a.adapters, 2),
                           dim3(kJoinWarps * 32), 0, st, (const int *)p.slot_id, (int)slots, (const float *)p.partial[0],
                           (const float *)p.partial[1], (T *)a.grad[0], (T *)a.grad[1], e0, e1));
  AB200_LAUNCH_CHECK();
}

bool rowsAlign(const void *p, long long ld, int width, int type) {
  const int size = type == DT_F32 ? 4 : 2;
  return p == nullptr || ((uintptr_t)p % 16 == 0 && ld * size % 16 == 0 && (long long)width * size % 16 == 0);
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
  case DT_F32:
    vec ? dispatchApply<float, true>(p, a.seg, stream) : dispatchApply<float, false>(p, a.seg, stream);
    break;
  case DT_F16:
    vec ? dispatchApply<__half, true>(p, a.seg, stream) : dispatchApply<__half, false>(p, a.seg, stream);
    break;
  default:
    vec ? dispatchApply<__nv_bfloat16, true>(p, a.seg, stream) : dispatchApply<__nv_bfloat16, false>(p, a.seg, stream);
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
