// Gradients of layer normalisation in one sweep over memory: dy, x (and residual) in, dx (and dresidual) out, and the sums of dy xhat and
// of dy for weight and bias on the way.
//   z = x or residual + dropout(x) again, xhat = (z - mean) rstd, g = dy w, dz = rstd (g - mean(g) - xhat mean(g xhat))
// A team of threads (norm.hpp) holds a row in registers; a thread owns the same columns of every row that its team works on, so the sums
// over rows are private registers until the workgroup's teams are added up through LDS and written as one partial sum
// [2][cols] a workgroup.  norm_finish adds the partial sums in a fixed order: no atomics, the same bits every time.
#include "norm.hpp"

namespace lbm {

#ifndef NB_U1
#define NB_U1 2
#define NB_U2 1
#define NB_G 1024
#define NB_GB 512
#endif

// dweight / dbias from the first partial sum when it is the only one
template <class T> __device__ __forceinline__ void put_sum(const NormArgs& a, int which, long long c, float v) {
  T* o = reinterpret_cast<T*>(which == 0 ? a.dweight : a.dbias);
  if (o != nullptr) o[c] = (T)v;
}
template <class TX> __device__ __forceinline__ void put_part(const NormArgs& a, int which, long long c, float v) {
  if (gridDim.x > 1) a.workspace[((long long)blockIdx.x * 2 + which) * a.cols + c] = v;
  else if (a.p_f32) put_sum<float>(a, which, c, v);
  else put_sum<TX>(a, which, c, v);
}

template <class TX, class TR, int RES, int K, int U, bool BLK>
__global__ __launch_bounds__(BLK ? 1024 : 256) void norm_bwd_kernel(NormArgs a, int shift) {
  __shared__ float red[BLK ? 64 : 4 * 512 * K];          // BLK: the row sums of two rows in turn; else: one sum of every wave, then of the other
  const int lanes = BLK ? blockDim.x : K > 1 ? 64 : 1 << shift;
  const int tl = BLK ? threadIdx.x : threadIdx.x & (lanes - 1);
  const int team = BLK ? 0 : K > 1 ? threadIdx.x >> 6 : threadIdx.x >> shift;
  const int teams = BLK ? 1 : K > 1 ? 4 : 256 >> shift;
  const int cols = (int)a.cols;
  const float inv = 1.0f / (float)cols;
  DropKey key{};
  if (RES) key = drop_key(a.drop);
  int nv[K];
  float w[K][8], dw[K][8] = {}, db[K][8] = {};
#pragma unroll
  for (int k = 0; k < K; ++k) {
    nv[k] = min(8, cols - (k * lanes + tl) * 8);
    load_param<TX>(a.weight, a.p_f32, (k * lanes + tl) * 8, nv[k], 1.0f, w[k]);
  }
  int par = 0;
  for (long long base = (long long)blockIdx.x * (teams * U); base < a.rows; base += (long long)gridDim.x * (teams * U)) {
    Vec8<TX> vx[U][K];
    Vec8<TR> vr[U][K], vd[U][K];
    float mean[U], rstd[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long row = base + u * teams + team;
      const bool in = row < a.rows;
      mean[u] = in ? a.mean[row] : 0.0f;
      rstd[u] = in ? a.rstd[row] : 0.0f;
#pragma unroll
      for (int k = 0; k < K; ++k) {       // past the row's end, and past the last row: zeros
        const int c = (k * lanes + tl) * 8, n = in ? nv[k] : 0;
        vd[u][k].load(reinterpret_cast<const TR*>(a.dy) + row * a.ld_dy + c, n);
        vx[u][k].load(reinterpret_cast<const TX*>(a.x) + row * a.ld_x + c, n);
        if (RES) vr[u][k].load(reinterpret_cast<const TR*>(a.residual) + row * a.ld_r + c, n);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long row = base + u * teams + team;
      float xh[K][8], s1 = 0.0f, s2 = 0.0f;
      uint32_t m[K];
#pragma unroll
      for (int k = 0; k < K; ++k) {
        m[k] = 0xffu;
        float scale = 1.0f;
        if (RES && a.drop.on) {
          m[k] = keep8((uint64_t)(row * a.cols + (k * lanes + tl) * 8), key, a.drop.tm1);
          scale = a.drop.scale;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float z = join_one<RES>(vx[u][k].get(j), RES ? vr[u][k].get(j) : 0.0f, m[k] >> j & 1, scale);
          xh[k][j] = (z - mean[u]) * rstd[u];
        }
        if (nv[k] < 8) {                  // nothing past the row's end may reach a sum (0 times an overflowed mean * rstd is no zero)
#pragma unroll
          for (int j = 0; j < 8; ++j) xh[k][j] = j < nv[k] ? xh[k][j] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float d = vd[u][k].get(j), g = d * w[k][j];
          s1 += g;
          s2 = fmaf(g, xh[k][j], s2);
          dw[k][j] = fmaf(d, xh[k][j], dw[k][j]);
          db[k][j] += d;
        }
      }
      if (BLK) {
        // one barrier a row: the next row writes the other half, and the one after it finds every thread past this row's reads
        s1 = wave64_sum(s1);
        s2 = wave64_sum(s2);
        float* sm = red + 32 * par;
        par ^= 1;
        if ((threadIdx.x & 63) == 0) {
          sm[2 * (threadIdx.x >> 6)] = s1;
          sm[2 * (threadIdx.x >> 6) + 1] = s2;
        }
        __syncthreads();
        s1 = s2 = 0.0f;
        for (int i = 0; i < (int)(blockDim.x >> 6); ++i) {
          s1 += sm[2 * i];
          s2 += sm[2 * i + 1];
        }
      } else {
        s1 = K > 1 ? wave64_sum(s1) : lanes_sum(s1, shift);
        s2 = K > 1 ? wave64_sum(s2) : lanes_sum(s2, shift);
      }
      const float c1 = s1 * inv, c2 = s2 * inv;
      if (row < a.rows) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (nv[k] <= 0) continue;
          const long long at = row * a.cols + (k * lanes + tl) * 8;
          float dz[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) dz[j] = rstd[u] * (fmaf(vd[u][k].get(j), w[k][j], -c1) - xh[k][j] * c2);
          if (RES && a.dresidual != nullptr) {
            Vec8<TR> o;
            o.set(dz);
            o.store(reinterpret_cast<TR*>(a.dresidual) + at, nv[k]);
          }
          if (a.dx != nullptr) {
            if (RES && a.drop.on) {
#pragma unroll
              for (int j = 0; j < 8; ++j) dz[j] = (m[k] >> j & 1) ? dz[j] * a.drop.scale : 0.0f;
            }
            Vec8<TX> o;
            o.set(dz);
            o.store(reinterpret_cast<TX*>(a.dx) + at, nv[k]);
          }
        }
      }
    }
  }
  if (a.dweight == nullptr && a.dbias == nullptr) return;
  if (BLK) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < nv[k]) {
          put_part<TX>(a, 0, (k * lanes + tl) * 8 + j, dw[k][j]);
          put_part<TX>(a, 1, (k * lanes + tl) * 8 + j, db[k][j]);
        }
    return;
  }
  // the teams of a wave, then the four waves
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float(&acc)[K][8] = which == 0 ? dw : db;
    if (K == 1) {
      for (int s = lanes; s < 64; s <<= 1)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[0][j] += __shfl_xor(acc[0][j], s);
    }
    if (which == 1) __syncthreads();
    const int wave = threadIdx.x >> 6;
    if ((int)(threadIdx.x & 63) < lanes) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) red[wave * (512 * K) + (k * lanes + tl) * 8 + j] = acc[k][j];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < cols; c += 256)
      put_part<TX>(a, which, c, (red[c] + red[512 * K + c]) + (red[2 * 512 * K + c] + red[3 * 512 * K + c]));
  }
}

// dweight / dbias = the partial sums added up in a fixed order: 32 columns x 32 slices of the partial sums a workgroup
template <class T>
__global__ __launch_bounds__(1024) void norm_finish_kernel(const float* part, int parts, long long cols, T* dweight, T* dbias) {
  __shared__ float sm[32][33];
  const int tc = threadIdx.x & 31, tg = threadIdx.x >> 5;
  const long long c = (long long)blockIdx.x * 32 + tc;              // over 2 cols: dweight, then dbias
  float s = 0.0f;
  if (c < 2 * cols) {
    const float* p = part + c;
#pragma unroll 8
    for (int g = tg; g < parts; g += 32) s += p[(long long)g * 2 * cols];
  }
  sm[tg][tc] = s;
  __syncthreads();
  if (tg < 1 && c < 2 * cols) {
    s = 0.0f;
#pragma unroll
    for (int g = 0; g < 32; ++g) s += sm[g][tc];
    T* o = c < cols ? dweight : dbias;
    if (o != nullptr) o[c < cols ? c : c - cols] = (T)s;
  }
}

int norm_finish(const NormArgs& a, int parts, hipStream_t s) {
  const unsigned grid = (unsigned)((2 * a.cols + 31) / 32);
  if (a.p_f32) norm_finish_kernel<float><<<grid, 1024, 0, s>>>(a.workspace, parts, a.cols, (float*)a.dweight, (float*)a.dbias);
  else if (a.x_type == kF16) norm_finish_kernel<_Float16><<<grid, 1024, 0, s>>>(a.workspace, parts, a.cols, (_Float16*)a.dweight, (_Float16*)a.dbias);
  else norm_finish_kernel<__bf16><<<grid, 1024, 0, s>>>(a.workspace, parts, a.cols, (__bf16*)a.dweight, (__bf16*)a.dbias);
  return check_launch("norm_backward");
}

static int rows_at_once(const NormShape& sh) { return sh.block ? 1 : sh.k == 1 ? NB_U1 : sh.k == 2 ? NB_U2 : 1; }
// workgroups = partial sums
static int norm_parts(long long rows, const NormShape& sh) {
  const long long per = (long long)sh.teams() * rows_at_once(sh);
  long long g = (rows + per - 1) / per;
  const long long most = sh.block ? NB_GB * 512 / sh.threads : NB_G;
  return (int)(g < 1 ? 1 : g < most ? g : most);
}

uint64_t norm_workspace_bytes(long long rows, long long cols) {
  const int parts = cols > kNormRowMax ? norm_wide_parts(rows, cols) : norm_parts(rows, norm_shape(cols));
  return (uint64_t)parts * 2 * (uint64_t)cols * sizeof(float);
}

template <class TX, class TR, int RES> static int backward(const NormArgs& a, hipStream_t s) {
  const NormShape sh = norm_shape(a.cols);
  const int grid = norm_parts(a.rows, sh);
  if (sh.block) norm_bwd_kernel<TX, TR, RES, 2, 1, true><<<grid, sh.threads, 0, s>>>(a, 0);
  else if (sh.k == 1) norm_bwd_kernel<TX, TR, RES, 1, NB_U1, false><<<grid, 256, 0, s>>>(a, sh.shift);
  else if (sh.k == 2) norm_bwd_kernel<TX, TR, RES, 2, NB_U2, false><<<grid, 256, 0, s>>>(a, 6);
  else norm_bwd_kernel<TX, TR, RES, 4, 1, false><<<grid, 256, 0, s>>>(a, 6);
  if (check_launch("norm_backward")) return -1;
  if (grid > 1 && (a.dweight != nullptr || a.dbias != nullptr)) return norm_finish(a, grid, s);
  return 0;
}

int norm_backward(const NormArgs& a, hipStream_t stream) {
  ProfScope prof("norm_backward", stream, 14.0 * a.rows * a.cols,
                 (double)a.rows * a.cols * (2.0 * elem_size(a.x_type) + elem_size(a.y_type) * (a.residual ? 3.0 : 1.0)));
  if (a.cols > kNormRowMax) return norm_wide_backward(a, stream);
  NORM_DISPATCH(backward, a, stream);
}

}  // namespace lbm
