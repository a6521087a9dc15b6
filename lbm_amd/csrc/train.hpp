// Operators of a training step around a block's residual join (transformer.py:272-338: norm(x + dropout(f(x)))): dropout from a
// counter-based generator and layer normalisation with its gradients.  Shared declarations and device helpers.
#pragma once
#include "common.hpp"

namespace lbm {

enum ElemType { kF32 = 0, kF16 = 1, kBF16 = 2 };   // LBM_TYPE_* of include/lbm_hip.h
inline int elem_size(int t) { return t == kF32 ? 4 : 2; }

// ---- dropout mask ------------------------------------------------------------------------------------------------
// Element e (row-major index in the logical tensor) lies in block e >> 3, slot e & 7.  W(n, part) = Philox4x32-10 of the counter
// (2 n + part, offset) under the key `seed`: four words = the upper (part 0) or lower (part 1) 16 bits of the 32-bit numbers of eight
// elements.  An element is kept where its number is above tm1 = round(p 2^32) - 1.  The upper halves decide all but one element in
// 65536, so the second evaluation is a rare branch: 32-bit probabilities at the price of 16-bit ones.
struct DropArgs {
  int on;                      // 0: p rounds to zero, nothing is dropped
  uint32_t tm1;                // keep where number > tm1 (0xffffffff: nothing is kept)
  float scale;                 // 2^32 / (2^32 - round(p 2^32)) = 1 / (1 - p) to 32 bits; 0 when nothing is kept
  uint64_t seed, offset;
  const uint64_t* seed_ptr;    // device word read in place of `seed` when not null (graph replays draw new masks)
};
int make_drop(double p, uint64_t seed, const void* seed_ptr, uint64_t offset, DropArgs& d);

struct DropKey { uint32_t k0, k1, o0, o1; };
__device__ __forceinline__ DropKey drop_key(const DropArgs& d) {
  uint64_t s = d.seed;
  if (d.seed_ptr != nullptr) s = *d.seed_ptr;
  return DropKey{(uint32_t)s, (uint32_t)(s >> 32), (uint32_t)d.offset, (uint32_t)(d.offset >> 32)};
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// Philox4x32 with ten rounds (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011)
__device__ __forceinline__ u32x4 philox(uint64_t n, DropKey k) {
  uint32_t c0 = (uint32_t)n, c1 = (uint32_t)(n >> 32), c2 = k.o0, c3 = k.o1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k.k0;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k.k1;
    c1 = (uint32_t)b;
    c3 = (uint32_t)a;
    k.k0 += 0x9E3779B9u;
    k.k1 += 0xBB67AE85u;
  }
  return u32x4{c0, c1, c2, c3};
}
// bit j: element 8 block + j is kept
__device__ __forceinline__ uint32_t block_keep(uint64_t block, const DropKey& k, uint32_t tm1) {
  const uint32_t th = tm1 >> 16, tl = tm1 & 0xffffu;
  const u32x4 w = philox(2 * block, k);
  uint32_t keep = 0;
  bool tie = false;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t h = (j & 1) ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu;
    keep |= h > th ? 1u << j : 0u;
    tie |= h == th;
  }
  if (tie) {
    const u32x4 l = philox(2 * block + 1, k);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t h = (j & 1) ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu;
      const uint32_t q = (j & 1) ? l[j >> 1] >> 16 : l[j >> 1] & 0xffffu;
      keep |= h == th && q > tl ? 1u << j : 0u;
    }
  }
  return keep;
}
// the same for eight elements that start anywhere: a row whose length is no multiple of eight straddles two blocks
__device__ __forceinline__ uint32_t keep8(uint64_t e, const DropKey& k, uint32_t tm1) {
  const uint32_t sh = (uint32_t)e & 7u;
  uint32_t m = block_keep(e >> 3, k, tm1);
  if (sh != 0) m = (m | block_keep((e >> 3) + 1, k, tm1) << 8) >> sh;
  return m;
}

// ---- eight consecutive elements of a row ---------------------------------------------------------------------------
// One 16-byte access (two for fp32) at any element alignment: gfx950 serves unaligned global accesses, an odd row length costs only the
// second cache line that some of them touch.  nv = how many of the eight exist (>= 8: all).
template <class T> struct Vec8;
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));
typedef u32x4 u32x4_a4 __attribute__((aligned(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

template <> struct Vec8<float> {
  u32x4 a, b;
  __device__ __forceinline__ void load(const float* p, int nv) {
    if (nv >= 8) {
      a = *reinterpret_cast<const u32x4_a4*>(p);
      b = *reinterpret_cast<const u32x4_a4*>(p + 4);
    } else {
      a = b = u32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < 7; ++j)
        if (j < nv) {
          const uint32_t w = __builtin_bit_cast(uint32_t, p[j]);
          if (j < 4) a[j & 3] = w;
          else b[j & 3] = w;
        }
    }
  }
  __device__ __forceinline__ void store(float* p, int nv) const {
    if (nv >= 8) {
      *reinterpret_cast<u32x4_a4*>(p) = a;
      *reinterpret_cast<u32x4_a4*>(p + 4) = b;
    } else {
#pragma unroll
      for (int j = 0; j < 7; ++j)
        if (j < nv) p[j] = __builtin_bit_cast(float, j < 4 ? a[j & 3] : b[j & 3]);
    }
  }
  __device__ __forceinline__ float get(int j) const { return __builtin_bit_cast(float, j < 4 ? a[j & 3] : b[j & 3]); }
  __device__ __forceinline__ void set(const float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      a[j] = __builtin_bit_cast(uint32_t, v[j]);
      b[j] = __builtin_bit_cast(uint32_t, v[j + 4]);
    }
  }
};
struct Vec8Half {       // f16 and bf16: eight elements in four words
  u32x4 a;
  __device__ __forceinline__ void load(const uint16_t* p, int nv) {
    if (nv >= 8) {
      a = *reinterpret_cast<const u32x4_a2*>(p);
    } else {
      a = u32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < 7; ++j)
        if (j < nv) a[j >> 1] |= (uint32_t)p[j] << (16 * (j & 1));
    }
  }
  __device__ __forceinline__ void store(uint16_t* p, int nv) const {
    if (nv >= 8) {
      *reinterpret_cast<u32x4_a2*>(p) = a;
    } else {
#pragma unroll
      for (int j = 0; j < 7; ++j)
        if (j < nv) p[j] = (uint16_t)(a[j >> 1] >> (16 * (j & 1)));
    }
  }
};
template <> struct Vec8<_Float16> : Vec8Half {
  __device__ __forceinline__ void load(const _Float16* p, int nv) { Vec8Half::load(reinterpret_cast<const uint16_t*>(p), nv); }
  __device__ __forceinline__ void store(_Float16* p, int nv) const { Vec8Half::store(reinterpret_cast<uint16_t*>(p), nv); }
  __device__ __forceinline__ float get(int j) const {
    const uint32_t w = a[j >> 1];      // a copy: __builtin_bit_cast of a vector's element to a vector reads the vector's first word
    return (float)__builtin_bit_cast(f16x2, w)[j & 1];
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {     // rounds to nearest even, beyond 65504 to infinity
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)v[2 * j], (_Float16)v[2 * j + 1]});
  }
};
template <> struct Vec8<__bf16> : Vec8Half {
  __device__ __forceinline__ void load(const __bf16* p, int nv) { Vec8Half::load(reinterpret_cast<const uint16_t*>(p), nv); }
  __device__ __forceinline__ void store(__bf16* p, int nv) const { Vec8Half::store(reinterpret_cast<uint16_t*>(p), nv); }
  __device__ __forceinline__ float get(int j) const {
    return __builtin_bit_cast(float, (j & 1) ? a[j >> 1] & 0xffff0000u : a[j >> 1] << 16);
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {     // v_cvt_pk_bf16_f32: nearest even
#pragma unroll
    for (int j = 0; j < 4; ++j)
      a[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{v[2 * j], v[2 * j + 1]}), bf16x2));
  }
};

// ---- arguments of layer_norm / dropout_add_layer_norm ----------------------------------------------------------------
struct NormArgs {
  const void* x;               // [rows, cols], row stride ld_x elements
  const void* residual;        // [rows, cols], row stride ld_r; null: plain layer normalisation
  const void* weight;          // [cols] or null (ones)
  const void* bias;            // [cols] or null (zeros)
  void* y;                     // [rows, cols] dense, type y_type
  float* mean;                 // [rows] or null (forward); read by the backward pass
  float* rstd;
  const void* dy;              // [rows, cols], row stride ld_dy, type y_type
  void* dx;                    // [rows, cols] dense, type x_type, or null
  void* dresidual;             // [rows, cols] dense, type y_type, or null
  void* dweight;               // [cols] or null
  void* dbias;                 // [cols] or null
  float* workspace;
  uint64_t workspace_bytes;
  long long rows, cols, ld_x, ld_r, ld_dy;
  int x_type, y_type;          // y_type = the residual's type (x_type without one)
  int p_f32;                   // weight / bias (and their gradients) are fp32, not x_type
  float eps;
  DropArgs drop;               // used only with a residual
};
int norm_forward(const NormArgs& a, hipStream_t stream);
int norm_backward(const NormArgs& a, hipStream_t stream);
uint64_t norm_workspace_bytes(long long rows, long long cols);
int dropout(const void* x, void* y, long long n, int type, const DropArgs& d, hipStream_t stream);

// weight / bias as fp32 (absent: `dflt`)
template <class TX> __device__ __forceinline__ void load_param(const void* p, int p_f32, long long c, int nv, float dflt, float (&v)[8]) {
  if (p == nullptr) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = dflt;
    return;
  }
  if (p_f32) {
    Vec8<float> r;
    r.load(reinterpret_cast<const float*>(p) + c, nv);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = r.get(j);
  } else {
    Vec8<TX> r;
    r.load(reinterpret_cast<const TX*>(p) + c, nv);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = r.get(j);
  }
}

// z = residual + dropout(x) for eight elements, the same expression in both passes.  A dropped element counts as zero whatever its
// value (a NaN or infinity that is dropped leaves no trace).
template <int RES> __device__ __forceinline__ float join_one(float x, float r, bool keep, float scale) {
  if (RES == 0) return x;
  return fmaf(keep ? x : 0.0f, scale, r);
}

// sum over the block's threads, the same value in every thread; `sm`: 16 floats that no earlier call still reads
__device__ __forceinline__ float block_sum(float v, float* sm) {
  v = wave_sum(v);
  const int nw = blockDim.x >> 6;
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = 0.0f;
  for (int i = 0; i < nw; ++i) t += sm[i];
  return t;
}

}  // namespace lbm
