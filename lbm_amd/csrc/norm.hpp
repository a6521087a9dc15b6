// Pieces that the layer-normalisation kernels share (norm_fwd.hip, norm_bwd.hip, norm_wide.hip).
#pragma once
#include "train.hpp"

namespace lbm {

constexpr long long kNormRowMax = 16384;      // longest row that a team holds in registers; beyond: norm_wide.hip

int norm_wide_forward(const NormArgs& a, hipStream_t stream);
int norm_wide_backward(const NormArgs& a, hipStream_t stream);
int norm_wide_parts(long long rows, long long cols);
int norm_finish(const NormArgs& a, int parts, hipStream_t stream);     // workspace [parts][2][cols] -> dweight, dbias

// ---- teams: the threads that share a row ------------------------------------------------------------------------------
// Thread tl of a team of T threads holds the 8-element chunks tl, T + tl, ... (K of them) of its row in registers.  Rows up to 1536
// columns (layer_norm's forward pass: 2048) belong to a power of two of lanes of one wave: of the pairs (T, K) with K <= 4 that hold the row the
// one with the fewest T * K chunks (a lane past the row's end costs as much as one inside), the larger T among equals, so that K = 4 is left
// for more than 192 chunks.  Longer rows belong to a workgroup.
struct NormShape {
  int k;            // chunks a thread
  int shift;        // log2 of the lanes of a team (rows of a wave)
  int threads;      // of a workgroup
  bool block;       // a team is a workgroup
  int teams() const { return block ? 1 : threads >> shift; }
};
inline NormShape norm_shape(long long cols, int most) {        // most: chunks that a wave may hold
  NormShape s{1, 0, 256, false};
  const int chunks = (int)((cols + 7) / 8);
  if (chunks > most) {
    s.block = true;
    s.k = 2;
    s.threads = (chunks + 127) / 128 * 64;
    return s;
  }
  int best = 1 << 30;
  for (int shift = 6; shift >= 0; --shift) {
    const int k = (chunks + (1 << shift) - 1) >> shift;
    if (k <= 4 && (k << shift) < best) {
      best = k << shift;
      s.k = k;
      s.shift = shift;
    }
  }
  return s;
}

// Where a chunk's eight elements are read: the last one of a row that is no multiple of eight is read from eight before the row's end on
// and cut, so no load lies outside of the row and none waits for a branch.  cut = 8: the chunk lies past the row's end.  (Rows of fewer
// than eight elements are a chunk that is loaded element by element, with cut = 8 - cols.)  Only a thread's last chunk can be cut: a team
// has no more chunks than it needs, (K - 1) T < ceil(cols / 8) for every shape above, so chunk k < K - 1 is whole and costs no test.
struct Span {
  int at, cut;
  __device__ __forceinline__ Span() {}
  __device__ __forceinline__ Span(int a, int c) : at(a), cut(c) {}
  template <LoadMode MODE> static __device__ __forceinline__ Span of(int c, int cols, bool last) {
    if (!last) return Span(c, 0);
    if (MODE == kShort) return Span(0, c == 0 ? 8 - cols : 8);
    const int at = min(c, cols - 8);
    return Span(at, min(c - at, 8));
  }
};
template <class TX, LoadMode MODE> __device__ __forceinline__ void load_param(const void* p, int p_f32, const Span& s, float dflt, float (&v)[8]) {
  if (p == nullptr) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = dflt;
  } else if (p_f32) {
    Vec8<float> r;
    r.template load<MODE>(reinterpret_cast<const float*>(p) + s.at, 8 - s.cut);
    r.template cut<MODE>(s.cut);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = r.get(j);
  } else {
    Vec8<TX> r;
    r.template load<MODE>(reinterpret_cast<const TX*>(p) + s.at, 8 - s.cut);
    r.template cut<MODE>(s.cut);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = r.get(j);
  }
}
// element offset of row r (below 2^32) at a stride below 2^31: one multiply
__device__ __forceinline__ uint64_t row_at(uint32_t r, uint32_t ld, int c) { return (uint64_t)r * ld + (uint32_t)c; }
// 1 / sqrt(v): v_rsq_f32 (1 ulp) and a Newton step in place of the correctly rounded square root and division (~25 instructions a row).  A variance
// beyond the range (infinite) gives NaN: no row of zeros that looks like a result.
__device__ __forceinline__ float rsqrt_newton(float v) {
  const float r = __builtin_amdgcn_rsqf(v);
  const float e = fmaf(-v * r, r, 1.0f);
  return fmaf(0.5f * r, e, r);
}

// The first mean m of a row is its sum times 1 / cols in fp32, off by some roundings of m: of no account beside the spread unless the row lies far from
// zero (1000 columns of 1000.1: 0.02 after the division by sqrt(eps)).  The second pass therefore sums the deviations z - m themselves beside their squares:
//   d = mean(z - m): the mean is m + d;   var = mean((z - m)^2) - d^2,   z - mean = (z - m) - d
// What is left grows with the spread and with e^2 |m| (e = 2^-24).  The difference of the squares and d^2 holds as long as the variance is not far below d^2;
// where it is (a constant row), it is rounding noise and 2^-18 of the squares stands for it, so that no eps makes a result of that noise.  The correction costs the
// forward pass 0 - 4 % (65536 x 256 f16 14.3 -> 14.9 us, 9000 x 16384 110 -> 113, 589824 x 256 none).
__device__ __forceinline__ float norm_variance(float squares, float d) {
  return fmaxf(fmaf(-d, d, squares), squares * 0x1p-18f);      // NaN and infinity come through the second
}

// a * b rounded by itself: contracted into the subtractions, m would be another number in z - m than in m + d
__device__ __forceinline__ float product(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

__device__ __forceinline__ float lane16_sum(float v) {     // v + the value 16 lanes away (lane ^ 16)
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
  const unsigned r0 = r[0], r1 = r[1];
  return __builtin_bit_cast(float, r0) + __builtin_bit_cast(float, r1);
}
__device__ __forceinline__ float lane32_sum(float v) {     // v + the value 32 lanes away
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
  const unsigned r0 = r[0], r1 = r[1];
  return __builtin_bit_cast(float, r0) + __builtin_bit_cast(float, r1);
}
// sum over aligned groups of 2^shift lanes, in every lane of the group
__device__ __forceinline__ float lanes_sum(float v, int shift) {
  if (shift >= 4) {
    v = row16_sum(v);
    if (shift >= 5) v = lane16_sum(v);
    if (shift >= 6) v = lane32_sum(v);
    return v;
  }
  for (int s = 1; s < 1 << shift; s <<= 1) v += __shfl_xor(v, s);
  return v;
}
// two sums in one go: a step of one fills the wait between two of the other
__device__ __forceinline__ void lanes_sum2(float& u, float& v, int shift) {
  if (shift >= 4) {
    u = row16_sum(u);
    v = row16_sum(v);
    if (shift >= 5) {
      u = lane16_sum(u);
      v = lane16_sum(v);
    }
    if (shift >= 6) {
      u = lane32_sum(u);
      v = lane32_sum(v);
    }
    return;
  }
  for (int s = 1; s < 1 << shift; s <<= 1) {
    u += __shfl_xor(u, s);
    v += __shfl_xor(v, s);
  }
}
// two sums behind one barrier; `sm`: 16 pairs
__device__ __forceinline__ void block_sum2(float& u, float& v, float (*sm)[2]) {
  lanes_sum2(u, v, 6);
  const int nw = blockDim.x >> 6;
  if ((threadIdx.x & 63) == 0) {
    sm[threadIdx.x >> 6][0] = u;
    sm[threadIdx.x >> 6][1] = v;
  }
  __syncthreads();
  u = v = 0.0f;
  for (int i = 0; i < nw; ++i) {
    u += sm[i][0];
    v += sm[i][1];
  }
}
__device__ __forceinline__ float wave64_sum(float v) { return lane32_sum(lane16_sum(row16_sum(v))); }

__device__ __forceinline__ u32x4 from_lane(const u32x4& v, int lane) {
  return u32x4{(uint32_t)__shfl((int)v[0], lane), (uint32_t)__shfl((int)v[1], lane), (uint32_t)__shfl((int)v[2], lane), (uint32_t)__shfl((int)v[3], lane)};
}
// The masks of a thread's K chunks; e0: the row's first element.  In a row whose length is no multiple of eight a chunk lies in two blocks,
// the second of which is the next chunk's first: it is fetched from the lane that drew it, and only behind a stripe's last lane one
// more is drawn.  BLK: a stripe (chunks k * lanes ...) runs over several waves, and lane k draws what lane 63 lacks of stripe k.
template <int K, bool BLK>
__device__ __forceinline__ void keep_row(Keep8 (&m)[K], uint64_t e0, const DropKey& key, uint32_t tm1, int cols, int lanes, int tl) {
  u32x4 w[K];
#pragma unroll
  for (int k = 0; k < K; ++k) w[k] = philox(2 * ((e0 >> 3) + (uint32_t)(k * lanes + tl)), key);
  if ((cols & 7) != 0) {
    const uint32_t sh = (uint32_t)e0 & 7u;
    const int seg = BLK ? 64 : lanes, self = threadIdx.x & 63, pos = self & (seg - 1), base = self - pos;
    u32x4 next[K];
#pragma unroll
    for (int k = 0; k < K; ++k) next[k] = from_lane(w[k], base + ((pos + 1) & (seg - 1)));
    if (BLK) {
      const u32x4 extra = philox(2 * ((e0 >> 3) + (uint32_t)((pos & 3) * lanes + tl - pos + 64)), key);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const u32x4 v = from_lane(extra, k);
        if (pos == 63) next[k] = v;
      }
    } else {
#pragma unroll
      for (int k = 0; k + 1 < K; ++k) {
        const u32x4 v = from_lane(w[k + 1], base);
        if (pos == lanes - 1) next[k] = v;
      }
      if (cols > (K * lanes - 1) * 8) {                    // the last lane's last chunk exists
        const u32x4 extra = philox(2 * ((e0 >> 3) + (uint32_t)(K * lanes)), key);
        if (pos == lanes - 1) next[K - 1] = extra;
      }
    }
    if (sh != 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) w[k] = straddle(w[k], next[k], sh);
    }
  }
#pragma unroll
  for (int k = 0; k < K; ++k) m[k] = keep_from(w[k], e0 + (uint32_t)((k * lanes + tl) * 8), key, tm1);
}

// May a half-precision row start in the middle of a dword?  Such rows are read dword by dword (Vec8, kOdd): 24995 x 6001 f16 forward 130 -> 126 us,
// backward 230 -> 189; 36612 x 4097 144 -> 117 and 258 -> 223; the join at 18312 x 8191 bf16 213 -> 174 and 369 -> 290, 73277 x 2047 209 -> 184 and 388 -> 309.
template <class T> inline bool odd_rows(const void* p, long long ld) { return sizeof(T) == 2 && ((ld & 1) != 0 || (reinterpret_cast<uintptr_t>(p) & 2) != 0); }

// calls f<TX, TR, RES>(a, s) for the types of a
#define NORM_DISPATCH(F, a, s)                                                                            \
  do {                                                                                                    \
    if (a.residual == nullptr) {                                                                          \
      if (a.x_type == kF32) return F<float, float, 0>(a, s);                                              \
      if (a.x_type == kF16) return F<_Float16, _Float16, 0>(a, s);                                        \
      return F<__bf16, __bf16, 0>(a, s);                                                                  \
    }                                                                                                     \
    if (a.x_type == kF32) return F<float, float, 1>(a, s);                                                \
    if (a.x_type == kF16) return a.y_type == kF32 ? F<_Float16, float, 1>(a, s) : F<_Float16, _Float16, 1>(a, s); \
    return a.y_type == kF32 ? F<__bf16, float, 1>(a, s) : F<__bf16, __bf16, 1>(a, s);                     \
  } while (0)

}  // namespace lbm
