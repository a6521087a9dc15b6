// Operators of a training step around a block's residual join (transformer.py:272-338: norm(x + dropout(f(x)))): dropout from a
// counter-based generator and layer normalisation with its gradients.  Shared declarations and device helpers.
#pragma once
#include "common.hpp"
#include "launch.hpp"

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
// Philox4x32 with ten rounds (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011).  A round is two
// v_mad_u64_u32 and two three-input exclusive ors; ten of them are what dropout computes, and stay below what it reads and writes.
__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) { return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96); }
__device__ __forceinline__ u32x4 philox(uint64_t n, DropKey k) {
  uint32_t c0 = (uint32_t)n, c1 = (uint32_t)(n >> 32), c2 = k.o0, c3 = k.o1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    c0 = xor3((uint32_t)(b >> 32), c1, k.k0);
    c2 = xor3((uint32_t)(a >> 32), c3, k.k1);
    c1 = (uint32_t)b;
    c3 = (uint32_t)a;
    k.k0 += 0x9E3779B9u;
    k.k1 += 0xBB67AE85u;
  }
  return u32x4{c0, c1, c2, c3};
}

// Eight elements' decisions: eight 16-bit numbers, an element is kept where its number is above `limit`.  Elements whose upper half
// ties with the threshold's are decided by the lower halves and then set to 0xffff or 0; limit is at most 0xfffe, so 0xffff is above it.
struct Keep8 {
  u32x4 w;
  __device__ __forceinline__ bool kept(int j, uint32_t limit) const {
    const uint32_t v = w[j >> 1];
    return (j & 1) ? v > (limit << 16 | 0xffffu) : (uint16_t)v > (uint16_t)limit;
  }
};
__device__ __forceinline__ uint32_t keep_limit(uint32_t tm1) { return min(tm1 >> 16, 0xfffeu); }

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pk_min(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
// does any of the eight halves equal the threshold's upper half?
__device__ __forceinline__ bool any_tie(const u32x4& w, uint32_t tm1) {
  const uint32_t hh = (tm1 >> 16) * 0x10001u;
  const uint32_t w0 = w[0] ^ hh, w1 = w[1] ^ hh, w2 = w[2] ^ hh, w3 = w[3] ^ hh;
  const uint32_t m = pk_min(pk_min(w0, w1), pk_min(w2, w3));
  return (m & 0xffffu) == 0 || m < 0x10000u;
}
__device__ __forceinline__ void settle_ties(u32x4& w, const u32x4& low, uint32_t tm1) {
  const uint32_t th = tm1 >> 16, tl = tm1 & 0xffffu;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t lo = w[i] & 0xffffu, hi = w[i] >> 16;
    if (lo == th) lo = (low[i] & 0xffffu) > tl ? 0xffffu : 0u;
    if (hi == th) hi = (low[i] >> 16) > tl ? 0xffffu : 0u;
    w[i] = hi << 16 | lo;
  }
}
__device__ __forceinline__ Keep8 block_keep(uint64_t block, const DropKey& k, uint32_t tm1) {
  Keep8 m{philox(2 * block, k)};
  if (any_tie(m.w, tm1)) settle_ties(m.w, philox(2 * block + 1, k), tm1);
  return m;
}
// eight 16-bit numbers from slot sh (1 .. 7) of block a on into block b
__device__ __forceinline__ u32x4 straddle(const u32x4& a, const u32x4& b, uint32_t sh) {
  u32x4 p = a, q = b;
  if (sh & 4) {
    p = u32x4{a[2], a[3], b[0], b[1]};
    q = u32x4{b[2], b[3], 0, 0};
  }
  if (sh & 2) {
    p = u32x4{p[1], p[2], p[3], q[0]};
    q[0] = q[1];
  }
  if (sh & 1) p = u32x4{p[0] >> 16 | p[1] << 16, p[1] >> 16 | p[2] << 16, p[2] >> 16 | p[3] << 16, p[3] >> 16 | q[0] << 16};
  return p;
}
// the eight elements from e on, `high` being the numbers' upper halves; rows whose length is no multiple of eight start anywhere in a block
__device__ __forceinline__ Keep8 keep_from(u32x4 high, uint64_t e, const DropKey& k, uint32_t tm1) {
  Keep8 m{high};
  if (any_tie(m.w, tm1)) {
    const uint32_t sh = (uint32_t)e & 7u;
    const uint64_t b = e >> 3;
    u32x4 low = philox(2 * b + 1, k);
    if (sh != 0) low = straddle(low, philox(2 * b + 3, k), sh);
    settle_ties(m.w, low, tm1);
  }
  return m;
}
__device__ __forceinline__ Keep8 keep8(uint64_t e, const DropKey& k, uint32_t tm1) {
  const uint32_t sh = (uint32_t)e & 7u;
  const uint64_t b = e >> 3;
  u32x4 high = philox(2 * b, k);
  if (sh != 0) high = straddle(high, philox(2 * b + 2, k), sh);
  return keep_from(high, e, k, tm1);
}

// ---- eight consecutive elements of a row ---------------------------------------------------------------------------
// One 16-byte access (two for fp32): gfx950 serves unaligned global accesses, at full rate where they start at a dword.
//   load           eight elements; near a row's end the caller reads earlier ones and cuts (below).  kOdd: half-precision rows that may start
//                  in the middle of a dword (6001 columns: 3.7 TB/s instead of 5.2 in the backward pass) are read from the dwords
//                  that hold them and shifted in cut; no dword without one of the eight is touched.  kShort: rows of n < 8 elements
//   load_some      the first nv of eight, element by element, and zeros
//   cut(s)         drops the first s elements and fills up with zeros (s = 8: all zeros); kShort: nothing but s = 8
//   store(p, nv)   the first nv of eight
enum LoadMode { kPlain, kOdd, kShort };
template <class T> struct Vec8;
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));
typedef u32x4 u32x4_a4 __attribute__((aligned(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_a2 __attribute__((aligned(2)));
typedef u32x2 u32x2_a4 __attribute__((aligned(4)));
typedef uint32_t u32_a2 __attribute__((aligned(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

template <> struct Vec8<float> {
  u32x4 a, b;
  template <LoadMode MODE = kPlain> __device__ __forceinline__ void load(const float* p, int n = 8) {
    if (MODE == kShort) {
      load_some(p, n);
      return;
    }
    a = *reinterpret_cast<const u32x4_a4*>(p);
    b = *reinterpret_cast<const u32x4_a4*>(p + 4);
  }
  __device__ __forceinline__ void load_some(const float* p, int nv) {
    a = b = u32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < nv) {
        const uint32_t w = __builtin_bit_cast(uint32_t, p[j]);
        if (j < 4) a[j & 3] = w;
        else b[j & 3] = w;
      }
  }
  template <LoadMode MODE = kPlain> __device__ __forceinline__ void cut(int s) {
    if (MODE == kShort) {
      if (s == 8) a = b = u32x4{0, 0, 0, 0};
      return;
    }
    if (s == 0) return;
    if (s & 4) { a = b; b = u32x4{0, 0, 0, 0}; }
    if (s & 2) { a = u32x4{a[2], a[3], b[0], b[1]}; b = u32x4{b[2], b[3], 0, 0}; }
    if (s & 1) { a = u32x4{a[1], a[2], a[3], b[0]}; b = u32x4{b[1], b[2], b[3], 0}; }
    if (s & 8) a = b = u32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ void store(float* p, int nv) const {
    if (nv >= 8) {
      *reinterpret_cast<u32x4_a4*>(p) = a;
      *reinterpret_cast<u32x4_a4*>(p + 4) = b;
      return;
    }
    if (nv & 4) *reinterpret_cast<u32x4_a4*>(p) = a;
    const u32x4 t = (nv & 4) ? b : a;
    p += nv & 4;
    if (nv & 2) *reinterpret_cast<u32x2_a4*>(p) = u32x2{t[0], t[1]};
    if (nv & 1) p[nv & 2] = __builtin_bit_cast(float, (nv & 2) ? (uint32_t)t[2] : (uint32_t)t[0]);
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
  uint32_t fifth, shift;          // kOdd only: the dword behind the four, and 0 or 16
  template <LoadMode MODE = kPlain> __device__ __forceinline__ void load(const void* p, int n = 8) {
    if (MODE == kShort) {
      load_some(p, n);
    } else if (MODE == kOdd) {
      const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(p) & 2u;
      const char* q = reinterpret_cast<const char*>(p) - off;
      a = *reinterpret_cast<const u32x4_a4*>(q);
      fifth = *reinterpret_cast<const uint32_t*>(q + 12 + 2 * off);      // off = 0: the fourth again
      shift = 8 * off;
    } else {
      a = *reinterpret_cast<const u32x4_a2*>(p);
    }
  }
  __device__ __forceinline__ void load_some(const void* q, int nv) {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(q);
    a = u32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < nv) a[j >> 1] |= (uint32_t)p[j] << (16 * (j & 1));
  }
  template <LoadMode MODE = kPlain> __device__ __forceinline__ void cut(int s) {
    if (MODE == kShort) {
      if (s == 8) a = u32x4{0, 0, 0, 0};
      return;
    }
    if (MODE == kOdd)
      a = u32x4{__builtin_amdgcn_alignbit(a[1], a[0], shift), __builtin_amdgcn_alignbit(a[2], a[1], shift), __builtin_amdgcn_alignbit(a[3], a[2], shift),
                __builtin_amdgcn_alignbit(fifth, a[3], shift)};
    if (s == 0) return;
    if (s & 4) a = u32x4{a[2], a[3], 0, 0};
    if (s & 2) a = u32x4{a[1], a[2], a[3], 0};
    if (s & 1) a = u32x4{a[0] >> 16 | a[1] << 16, a[1] >> 16 | a[2] << 16, a[2] >> 16 | a[3] << 16, a[3] >> 16};
    if (s & 8) a = u32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ void store(void* q, int nv) const {
    uint16_t* p = reinterpret_cast<uint16_t*>(q);
    if (nv >= 8) {
      *reinterpret_cast<u32x4_a2*>(p) = a;
      return;
    }
    if (nv & 4) *reinterpret_cast<u32x2_a2*>(p) = u32x2{a[0], a[1]};
    const u32x2 t = (nv & 4) ? u32x2{a[2], a[3]} : u32x2{a[0], a[1]};
    p += nv & 4;
    if (nv & 2) *reinterpret_cast<u32_a2*>(p) = t[0];
    if (nv & 1) p[nv & 2] = (uint16_t)((nv & 2) ? t[1] : t[0]);
  }
};
template <> struct Vec8<_Float16> : Vec8Half {
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
  __device__ __forceinline__ float get(int j) const {
    const uint32_t w = a[j >> 1];
    return __builtin_bit_cast(float, (j & 1) ? w & 0xffff0000u : w << 16);
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
