// Device helpers of the digital operators: element types, a warp's span of 256 neighbouring
// elements of a row, and the counter-based keep decision of the dropout.
#pragma once

#include "common.cuh"
#include "digital.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace ab200 {

// streaming multiprocessors of the current device
int digitalSmCount();

enum : uint32_t {
  TAG_DROPOUT = 0xB0000000u,     // high half-words of the draws
  TAG_DROPOUT_LOW = 0xB0000001u, // low half-words, looked at only where a high one ties
};

template <typename T> struct Elem;
template <> struct Elem<float> {
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <> struct Elem<__half> {
  static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};
template <> struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};

// two 16-bit elements of one word
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// ---- spans ------------------------------------------------------------------------------------
// A warp works on spans of 256 neighbouring elements of a row, eight per lane. Where every row
// starts on the width of eight elements and the width is a multiple of eight (VEC), a lane has
// eight neighbours, one 16-byte (16-bit types) or 32-byte (fp32, the widest load of this GPU)
// access; elsewhere lane l has the elements l, l + 32, ..., so that single loads stay coalesced.
// col(i) is the column of a lane's element i in both.
template <bool VEC> struct Span {
  static __device__ __forceinline__ int col(int span, int lane, int i) {
    return span * 256 + (VEC ? lane * 8 + i : lane + i * 32);
  }
};

__device__ __forceinline__ void load32B(const float *p, float v[8]) {
  asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
                 "=f"(v[7])
               : "l"(p));
}
__device__ __forceinline__ void store32B(float *p, const float v[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(v[0]), "f"(v[1]),
               "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}
template <typename T> __device__ __forceinline__ void unpack8(const uint4 &q, float v[8]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 f = unpack2<T>(w[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// the eight elements of a lane as they lie in memory, so that loads can be issued long before the
// conversion; columns past the end read as zero
template <typename T, bool VEC> struct Raw8 {
  uint4 q;
  __device__ __forceinline__ void load(const T *row, int span, int lane, int cols) {
    q = make_uint4(0, 0, 0, 0);
    if (VEC) {
      const int c = Span<true>::col(span, lane, 0);
      if (c < cols) {
        q = *reinterpret_cast<const uint4 *>(row + c);
      }
    } else {
      uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int c = Span<false>::col(span, lane, i);
        if (c < cols) {
          const uint32_t b = reinterpret_cast<const uint16_t *>(row)[c];
          w[i >> 1] |= b << (16 * (i & 1));
        }
      }
      q = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  __device__ __forceinline__ void get(float v[8]) const { unpack8<T>(q, v); }
  // elements whose half of the masks is zero become zero, whatever they were
  __device__ __forceinline__ void mask(const uint32_t m[4]) {
    q = make_uint4(q.x & m[0], q.y & m[1], q.z & m[2], q.w & m[3]);
  }
};
template <bool VEC> struct Raw8<float, VEC> {
  float f[8];
  __device__ __forceinline__ void load(const float *row, int span, int lane, int cols) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      f[i] = 0.0f;
    }
    if (VEC) {
      const int c = Span<true>::col(span, lane, 0);
      if (c < cols) {
        load32B(row + c, f);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int c = Span<false>::col(span, lane, i);
        if (c < cols) {
          f[i] = row[c];
        }
      }
    }
  }
  __device__ __forceinline__ void get(float v[8]) const {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      v[i] = f[i];
    }
  }
};

template <typename T, bool VEC>
__device__ __forceinline__ void storeSpan(T *row, int span, int lane, int cols, const float v[8]) {
  if (VEC) {
    const int c = Span<true>::col(span, lane, 0);
    if (c < cols) {
      if constexpr (sizeof(T) == 4) {
        store32B(reinterpret_cast<float *>(row) + c, v);
      } else {
        uint4 q;
        q.x = pack2<T>(v[0], v[1]);
        q.y = pack2<T>(v[2], v[3]);
        q.z = pack2<T>(v[4], v[5]);
        q.w = pack2<T>(v[6], v[7]);
        *reinterpret_cast<uint4 *>(row + c) = q;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int c = Span<false>::col(span, lane, i);
      if (c < cols) {
        row[c] = Elem<T>::put(v[i]);
      }
    }
  }
}

// ---- rows ahead -------------------------------------------------------------------------------
// A kernel that walks over 16-bit rows fetches the next one with cp.async while it works on the present one:
// every thread copies the elements that it will read itself into slots of its own, so no barrier and
// no wait on other threads is needed, and the registers stay free. Two stages; a stage has a slot of 16 bytes
// per tensor, span and thread, threads side by side.
template <typename T, int NS> struct RowRing {
  const unsigned char *own; // this thread's first slot
  int plane;                // bytes from slot to slot
  int per_stage;            // slots
  __device__ __forceinline__ RowRing(const void *smem, int tensors) {
    own = (const unsigned char *)smem + threadIdx.x * 16;
    plane = blockDim.x * 16;
    per_stage = tensors * NS;
  }
  static size_t bytes(int tensors, int threads) { return (size_t)2 * tensors * NS * 16 * threads; }
  __device__ __forceinline__ int slot(int stage, int tensor, int s) const {
    return (stage * per_stage + tensor * NS + s) * plane;
  }
  // columns past the end become zeros, without a read
  __device__ __forceinline__ void issue(int stage, int tensor, int s, const T *row, int span, int lane, int cols) const {
    const int c = Span<true>::col(span, lane, 0);
    const uint32_t dst = (uint32_t)__cvta_generic_to_shared(own + slot(stage, tensor, s));
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(row + c), "r"(c < cols ? 16 : 0)
                 : "memory");
  }
  static __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
  // all but the newest group of this thread have arrived
  static __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }
  __device__ __forceinline__ void get(int stage, int tensor, int s, Raw8<T, true> &r) const {
    r.q = *reinterpret_cast<const uint4 *>(own + slot(stage, tensor, s));
  }
};

// pairs of 16-bit results, masked as above
template <typename T>
__device__ __forceinline__ void storeMasked(T *row, int span, int lane, int cols, const float v[8], const uint32_t m[4]) {
  const int c = Span<true>::col(span, lane, 0);
  if (c < cols) {
    *reinterpret_cast<uint4 *>(row + c) = make_uint4(pack2<T>(v[0], v[1]) & m[0], pack2<T>(v[2], v[3]) & m[1],
                                                     pack2<T>(v[4], v[5]) & m[2], pack2<T>(v[6], v[7]) & m[3]);
  }
}

// ---- dropout ----------------------------------------------------------------------------------
// Element (row, col) is kept when a 32-bit word of its own is at least p * 2^32. The word's high
// half is lane col % 8 of the Philox4x32-10 block (row * ceil(cols / 8) + col / 8), its low half
// the same lane of a second block (TAG_DROPOUT_LOW), so one draw serves eight elements; the second
// one is made only where a high half equals the threshold's (once in 2^13 blocks), which keeps the
// probability exact to 2^-32 at half the draws that one word per element would take.
//
// The decision is taken two half-words at a time: bit 15 and bit 31 of a word of Kept say whether
// its two elements stay, and a byte permutation spreads them into masks. With 16-bit rows the whole
// GPU's integer pipe is what a dropout costs (Philox and 8 comparisons one by one: 75 % of that pipe, 80 us at
// 16384 x 4096 bf16), so every instruction here shows.
struct DropKey {
  uint32_t hi2; // the high half of the threshold, twice
  uint32_t lo;  // its low half; 65536 (with hi 65535) where everything is dropped
  float scale;  // 1 / (1 - p)
  uint32_t call;
  uint32_t a[10], b[10]; // Philox's keys of the ten rounds, which instructions take from constant memory
};
inline DropKey dropKey(const DropoutArgs &d) {
  const uint64_t thr = (uint64_t)(d.p * 4294967296.0 + 0.5);
  const bool all = thr >> 32 != 0;
  const uint32_t hi = all ? 0xffffu : (uint32_t)(thr >> 16);
  DropKey k;
  k.hi2 = hi | hi << 16;
  k.lo = all ? 0x10000u : (uint32_t)(thr & 0xffffu);
  k.scale = d.p < 1.0 ? (float)(1.0 / (1.0 - d.p)) : 0.0f;
  k.call = d.call;
  for (uint32_t r = 0; r < 10; r++) {
    k.a[r] = (uint32_t)d.seed + r * 0x9E3779B9u;
    k.b[r] = (uint32_t)(d.seed >> 32) + r * 0xBB67AE85u;
  }
  return k;
}
__device__ __forceinline__ void dropWords(const DropKey &k, uint64_t block, uint32_t tag, uint32_t out[4]) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = k.call, c3 = tag;
#pragma unroll
  for (int r = 0; r < 10; r++) { // philox4x32_10 with the keys at hand
    const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k.a[r];
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k.b[r];
    c1 = (uint32_t)p1;
    c3 = (uint32_t)p0;
  }
  out[0] = c0;
  out[1] = c1;
  out[2] = c2;
  out[3] = c3;
}
// Bits 15 and 31 of word i: half-words 0 and 1 of the block's word i (elements 2 i and 2 i + 1) stay;
// the other bits mean nothing.
struct Kept {
  uint32_t w[4];
};
__device__ __forceinline__ Kept keepBlock(const DropKey &k, uint64_t block) {
  constexpr uint32_t H = 0x80008000u;
  uint32_t w[4];
  dropWords(k, block, TAG_DROPOUT, w);
  Kept kept;
  uint32_t differ[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    // unsigned w >= hi in each half: the low 15 bits by a subtraction that cannot borrow from the
    // other half, the top bits where they differ
    const uint32_t low = (w[i] | H) - (k.hi2 & ~H);
    differ[i] = w[i] ^ k.hi2;
    kept.w[i] = (w[i] & ~k.hi2) | (~differ[i] & low);
  }
  // a half-word of `differ` that is zero is a tie (the borrow of one may name the other's as well)
  uint32_t tie = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    tie |= (differ[i] - 0x00010001u) & ~differ[i];
  }
  if ((tie & H) != 0 && k.lo != 0) {
    uint32_t l[4];
    dropWords(k, block, TAG_DROPOUT_LOW, l);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if ((differ[i] & 0xffffu) == 0 && (l[i] & 0xffffu) < k.lo) {
        kept.w[i] &= ~0x8000u;
      }
      if (differ[i] >> 16 == 0 && l[i] >> 16 < k.lo) {
        kept.w[i] &= ~0x80000000u;
      }
    }
  }
  return kept;
}
// byte selectors with their top bit set repeat the sign of the byte (the CUDA intrinsic drops that bit)
__device__ __forceinline__ uint32_t signMask(uint32_t w, uint32_t selectors) {
  uint32_t m;
  asm("prmt.b32 %0, %1, %1, %2;" : "=r"(m) : "r"(w), "r"(selectors));
  return m;
}
// The same for the elements that a lane holds of a span. Every lane of the warp draws the block of
// its own eight neighbours; without VEC the bits are passed to the lanes that hold the elements, and
// element i of a lane is again bit 15 (i even) or 31 of word i / 2. All lanes have to call it.
template <bool VEC>
__device__ __forceinline__ Kept keepOfSpan(const DropKey &k, long long row, int span, int lane, int cols) {
  const uint64_t blocks = (uint64_t)((cols + 7) >> 3);
  Kept mine = keepBlock(k, (uint64_t)row * blocks + (uint64_t)(span * 32 + lane));
  if (!VEC) {
    constexpr uint32_t H = 0x80008000u;
    // half-word j of the block at bit 12 + j / 2 + 16 (j odd)
    const uint32_t all = ((mine.w[0] & H) >> 3) | ((mine.w[1] & H) >> 2) | ((mine.w[2] & H) >> 1) | (mine.w[3] & H);
    const int at = 12 + ((lane & 7) >> 1) + 16 * (lane & 1);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint32_t b = (__shfl_sync(0xffffffffu, all, (lane >> 3) + 4 * i) >> at) & 1u;
      mine.w[i >> 1] = (i & 1) ? mine.w[i >> 1] | b << 31 : b << 15;
    }
  }
  return mine;
}
// masks of the pairs of 16-bit elements: a quarter of the masks of eight floats
__device__ __forceinline__ void pairMasks(const Kept &kept, uint32_t m[4]) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    m[i] = signMask(kept.w[i], 0xbb99);
  }
}
// v = kept ? v * scale : 0, whatever v is
__device__ __forceinline__ void dropSpan(const DropKey &k, const Kept &kept, float v[8]) {
#pragma unroll
  for (int i = 0; i < 8; i++) {
    // the bit, 32 times
    const uint32_t mask = signMask(kept.w[i >> 1], (i & 1) ? 0xbbbb : 0x9999);
    v[i] = __uint_as_float(__float_as_uint(v[i] * k.scale) & mask);
  }
}

// rows and width fit the accesses of eight elements
inline bool spansAlign(const void *p, long long ld, int type) {
  const uintptr_t bytes = type == DT_F32 ? 32 : 16;
  return p == nullptr || ((uintptr_t)p % bytes == 0 && ld % 8 == 0);
}

} // namespace ab200
