// Layer normalisation with the row in registers: y = (z - mean) rstd w + b, z = x or residual + dropout(x).
// One sweep over memory: a team of threads (norm.hpp) loads its row, sums it, sums the squared deviations from that mean (the two-pass
// form: no cancellation however large the mean) and writes y.  Bound by HBM: x (and residual) in, y out.  U rows a team are loaded before
// the first is used, and a workgroup ends after them: a grid in row order keeps the whole chip on neighbouring pages.
#include "norm.hpp"

namespace lbm {

template <class TX, class TR, int RES, int K, int U, bool BLK>
__global__ __launch_bounds__(BLK ? 1024 : 256) void norm_fwd_kernel(NormArgs a, int shift) {
  __shared__ float sm[2][16];
  const int lanes = BLK ? blockDim.x : K > 1 ? 64 : 1 << shift;
  const int tl = BLK ? threadIdx.x : threadIdx.x & (lanes - 1);
  const int team = BLK ? 0 : K > 1 ? threadIdx.x >> 6 : threadIdx.x >> shift;
  const int teams = BLK ? 1 : K > 1 ? 4 : 256 >> shift;
  const int cols = (int)a.cols;
  const float inv = 1.0f / (float)cols;
  DropKey key{};
  if (RES) key = drop_key(a.drop);
  int nv[K];
#pragma unroll
  for (int k = 0; k < K; ++k) nv[k] = min(8, cols - (k * lanes + tl) * 8);
  for (long long base = (long long)blockIdx.x * (teams * U); base < a.rows; base += (long long)gridDim.x * (teams * U)) {
    Vec8<TX> vx[U][K];
    Vec8<TR> vr[U][K];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long row = base + u * teams + team;
      const bool in = row < a.rows;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (k * lanes + tl) * 8, n = in ? nv[k] : 0;
        vx[u][k].load(reinterpret_cast<const TX*>(a.x) + row * a.ld_x + c, n);
        if (RES) vr[u][k].load(reinterpret_cast<const TR*>(a.residual) + row * a.ld_r + c, n);
      }
    }
    float w[K][8], b[K][8];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      load_param<TX>(a.weight, a.p_f32, (k * lanes + tl) * 8, nv[k], 1.0f, w[k]);
      load_param<TX>(a.bias, a.p_f32, (k * lanes + tl) * 8, nv[k], 0.0f, b[k]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long row = base + u * teams + team;
      float z[K][8], s = 0.0f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        uint32_t m = 0xffu;
        float scale = 1.0f;
        if (RES && a.drop.on) {
          m = keep8((uint64_t)(row * a.cols + (k * lanes + tl) * 8), key, a.drop.tm1);
          scale = a.drop.scale;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          z[k][j] = join_one<RES>(vx[u][k].get(j), RES ? vr[u][k].get(j) : 0.0f, m >> j & 1, scale);
          s += z[k][j];                                    // elements past the row's end were loaded as zeros
        }
      }
      const float mean = (BLK ? block_sum(s, sm[0]) : K > 1 ? wave64_sum(s) : lanes_sum(s, shift)) * inv;
      s = 0.0f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int j = 0; j < 8; ++j) z[k][j] -= mean;
        if (nv[k] < 8) {
#pragma unroll
          for (int j = 0; j < 8; ++j) z[k][j] = j < nv[k] ? z[k][j] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) s = fmaf(z[k][j], z[k][j], s);
      }
      const float var = (BLK ? block_sum(s, sm[1]) : K > 1 ? wave64_sum(s) : lanes_sum(s, shift)) * inv;
      const float rstd = 1.0f / sqrtf(var + a.eps);
      if (row < a.rows) {
        if (tl == 0 && a.mean != nullptr) {
          a.mean[row] = mean;
          a.rstd[row] = rstd;
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (nv[k] <= 0) continue;
#pragma unroll
          for (int j = 0; j < 8; ++j) z[k][j] = fmaf(z[k][j] * rstd, w[k][j], b[k][j]);
          Vec8<TR> o;
          o.set(z[k]);
          o.store(reinterpret_cast<TR*>(a.y) + row * a.cols + (k * lanes + tl) * 8, nv[k]);
        }
      }
    }
  }
}

#ifndef NF_U1
#define NF_U1 2
#define NF_U2 1
#endif
template <class TX, class TR, int RES> static int forward(const NormArgs& a, hipStream_t s) {
  const NormShape sh = norm_shape(a.cols);
  const int u = sh.block ? 1 : sh.k == 1 ? NF_U1 : sh.k == 2 ? NF_U2 : 1;
  const long long per = (long long)sh.teams() * u, want = (a.rows + per - 1) / per;
  const unsigned grid = (unsigned)(want < (1ll << 30) ? want : (1ll << 30));
  if (sh.block) norm_fwd_kernel<TX, TR, RES, 2, 1, true><<<grid, sh.threads, 0, s>>>(a, 0);
  else if (sh.k == 1) norm_fwd_kernel<TX, TR, RES, 1, NF_U1, false><<<grid, 256, 0, s>>>(a, sh.shift);
  else if (sh.k == 2) norm_fwd_kernel<TX, TR, RES, 2, NF_U2, false><<<grid, 256, 0, s>>>(a, 6);
  else norm_fwd_kernel<TX, TR, RES, 4, 1, false><<<grid, 256, 0, s>>>(a, 6);
  return check_launch("norm_forward");
}

int norm_forward(const NormArgs& a, hipStream_t stream) {
  if (a.rows == 0) return 0;
  ProfScope prof("norm_forward", stream, 8.0 * a.rows * a.cols,
                 (double)a.rows * a.cols * (elem_size(a.x_type) + elem_size(a.y_type) * (a.residual ? 2.0 : 1.0)));
  if (a.cols > kNormRowMax) return norm_wide_forward(a, stream);
  NORM_DISPATCH(forward, a, stream);
}

}  // namespace lbm
