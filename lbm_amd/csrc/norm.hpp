// Pieces that the layer-normalisation kernels share (norm_fwd.hip, norm_bwd.hip, norm_wide.hip).
#pragma once
#include "train.hpp"

namespace lbm {

constexpr long long kNormRowMax = 16384;      // longest row that a workgroup holds in registers; beyond: norm_wide.hip

int norm_wide_forward(const NormArgs& a, hipStream_t stream);
int norm_wide_backward(const NormArgs& a, hipStream_t stream);
int norm_wide_parts(long long rows, long long cols);
int norm_finish(const NormArgs& a, int parts, hipStream_t stream);     // workspace [parts][2][cols] -> dweight, dbias

// the eight z values of a chunk, and the mask bits when something is dropped
template <class TX, class TR, int RES>
__device__ __forceinline__ uint32_t load_z(const NormArgs& a, const DropKey& key, long long row, long long c, int nv, float (&z)[8]) {
  Vec8<TX> vx;
  vx.load(reinterpret_cast<const TX*>(a.x) + row * a.ld_x + c, nv);
  uint32_t m = 0xffu;
  Vec8<TR> vr;
  float scale = 1.0f;
  if (RES) {
    vr.load(reinterpret_cast<const TR*>(a.residual) + row * a.ld_r + c, nv);
    if (a.drop.on) {
      m = keep8((uint64_t)(row * a.cols + c), key, a.drop.tm1);
      scale = a.drop.scale;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) z[j] = join_one<RES>(vx.get(j), RES ? vr.get(j) : 0.0f, m >> j & 1, scale);
  return m;
}

// ---- teams: the threads that share a row ------------------------------------------------------------------------------
// Thread tl of a team of T holds the 8-element chunks tl, T + tl, ... (K of them) of its row in registers.  Up to 512 columns a team is a
// power of two of lanes (a wave works on several short rows), up to 2048 a wave with K = 2 or 4 chunks a lane, beyond a workgroup.
struct NormShape {
  int k;            // chunks a thread
  int shift;        // log2 of the lanes of a team (wave teams)
  int threads;      // of a workgroup
  bool block;       // a team is a workgroup
  int teams() const { return block ? 1 : threads >> shift; }
};
inline NormShape norm_shape(long long cols) {
  NormShape s{1, 0, 256, false};
  const int chunks = (int)((cols + 7) / 8);
  if (cols <= 2048) {
    while (s.shift < 6 && (1 << s.shift) < chunks) ++s.shift;
    s.k = chunks <= 64 ? 1 : chunks <= 128 ? 2 : 4;
  } else {
    s.block = true;
    s.k = 2;
    s.threads = (chunks + 127) / 128 * 64;
  }
  return s;
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
__device__ __forceinline__ float wave64_sum(float v) { return lane32_sum(lane16_sum(row16_sum(v))); }

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
