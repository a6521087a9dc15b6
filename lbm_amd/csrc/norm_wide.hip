// Layer normalisation of rows beyond what a workgroup holds in registers, of any length, forward and backward: a workgroup walks a row in
// several sweeps (the later ones find it in L2) and the gradients of weight and bias are summed by a kernel of their own that owns
// columns.  8000 x 20000 bf16 210 us forward (3.0 TB/s of x and y), 416 us backward (2.3), the join 332 and 666 (2.9, 2.4): three sweeps over a row
// instead of one.
//   z = residual + dropout(x);  m = mean(z);  v = mean((z - m)^2) (norm_variance);  rstd = 1 / sqrt(v + eps);  xhat = (z - m) rstd;  y = xhat w + b
//   g = dy w;  dz = rstd (g - mean(g) - xhat mean(g xhat));  dresidual = dz;  dx = keep ? dz scale : 0
//   dw = sum over rows of dy xhat;  db = sum over rows of dy
// Sums of eight are fp32, a thread's chunks of a row add up in fp64 (a row may have 2^28 columns, 2^17 chunks a thread), threads in fp32.  z is rebuilt from x, residual and the mask in the backward pass: storing it would move the same bytes (one write
// and one read against two reads for one), round it, and hold one more tensor.
#include "norm.hpp"

namespace lbm {

template <class T> __device__ __forceinline__ void load_nv(Vec8<T>& v, const T* p, int nv) {
  if (nv == 8) v.load(p);
  else v.load_some(p, nv);
}
// weight / bias as fp32 (absent: `dflt`)
template <class TX> __device__ __forceinline__ void load_param_some(const void* p, int p_f32, long long c, int nv, float dflt, float (&v)[8]) {
  Vec8<float> f;
  Vec8<TX> h;
  if (p != nullptr) {
    if (p_f32) load_nv(f, reinterpret_cast<const float*>(p) + c, nv);
    else load_nv(h, reinterpret_cast<const TX*>(p) + c, nv);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = p == nullptr ? dflt : p_f32 ? f.get(j) : h.get(j);
}
// the eight z values of a chunk; true where something may be dropped (then m says which)
template <class TX, class TR, int RES>
__device__ __forceinline__ bool load_z(const NormArgs& a, const DropKey& key, long long row, long long c, int nv, float (&z)[8], Keep8& m) {
  Vec8<TX> vx;
  Vec8<TR> vr;
  load_nv(vx, reinterpret_cast<const TX*>(a.x) + row * a.ld_x + c, nv);
  if (RES) load_nv(vr, reinterpret_cast<const TR*>(a.residual) + row * a.ld_r + c, nv);
  const bool drop = RES && a.drop.on;
  if (drop) m = keep8((uint64_t)(row * a.cols + c), key, a.drop.tm1);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    z[j] = join_one<RES>(vx.get(j), RES ? vr.get(j) : 0.0f, !drop || m.kept(j, keep_limit(a.drop.tm1)), drop ? a.drop.scale : 1.0f);
  return drop;
}

template <class TX, class TR, int RES>
__global__ __launch_bounds__(256) void norm_wide_fwd_kernel(NormArgs a) {
  __shared__ float sm[16], sm2[16][2];
  DropKey key{};
  if (RES) key = drop_key(a.drop);
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    double s64 = 0.0, d64 = 0.0;              // a thread's chunks add up in 64 bits
    float z[8];
    Keep8 m;
    for (long long c = threadIdx.x * 8; c < a.cols; c += 2048) {
      const int nv = (int)min(8ll, a.cols - c);
      load_z<TX, TR, RES>(a, key, row, c, nv, z, m);
      float t = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) t += j < nv ? z[j] : 0.0f;
      s64 += t;
    }
    const float mean = block_sum((float)s64, sm) / (float)a.cols;
    s64 = 0.0;
    for (long long c = threadIdx.x * 8; c < a.cols; c += 2048) {
      const int nv = (int)min(8ll, a.cols - c);
      load_z<TX, TR, RES>(a, key, row, c, nv, z, m);
      float t = 0.0f, u = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        t += j < nv ? (z[j] - mean) * (z[j] - mean) : 0.0f;
        u += j < nv ? z[j] - mean : 0.0f;
      }
      s64 += t;
      d64 += u;
    }
    float s = (float)s64, d = (float)d64;
    block_sum2(s, d, sm2);
    d /= (float)a.cols;                       // corrects the mean (norm.hpp)
    const float rstd = rsqrt_newton(norm_variance(s / (float)a.cols, d) + a.eps);
    if (threadIdx.x == 0 && a.mean != nullptr) {
      a.mean[row] = mean + d;
      a.rstd[row] = rstd;
    }
    for (long long c = threadIdx.x * 8; c < a.cols; c += 2048) {
      const int nv = (int)min(8ll, a.cols - c);
      float w[8], b[8];
      load_z<TX, TR, RES>(a, key, row, c, nv, z, m);
      load_param_some<TX>(a.weight, a.p_f32, c, nv, 1.0f, w);
      load_param_some<TX>(a.bias, a.p_f32, c, nv, 0.0f, b);
#pragma unroll
      for (int j = 0; j < 8; ++j) z[j] = fmaf((z[j] - mean - d) * rstd, w[j], b[j]);
      Vec8<TR> o;
      o.set(z);
      o.store(reinterpret_cast<TR*>(a.y) + row * a.cols + c, nv);
    }
  }
}

template <class TX, class TR, int RES>
__global__ __launch_bounds__(256) void norm_wide_dx_kernel(NormArgs a) {
  __shared__ float sm[2][16];
  DropKey key{};
  if (RES) key = drop_key(a.drop);
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float mean = a.mean[row], rstd = a.rstd[row];
    double s1 = 0.0, s2 = 0.0;
    float z[8], w[8];
    Keep8 m;
    for (long long c = threadIdx.x * 8; c < a.cols; c += 2048) {
      const int nv = (int)min(8ll, a.cols - c);
      load_z<TX, TR, RES>(a, key, row, c, nv, z, m);
      load_param_some<TX>(a.weight, a.p_f32, c, nv, 1.0f, w);
      Vec8<TR> d;
      load_nv(d, reinterpret_cast<const TR*>(a.dy) + row * a.ld_dy + c, nv);
      float t = 0.0f, u = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float g = d.get(j) * w[j];
        t += j < nv ? g : 0.0f;
        u += j < nv ? g * ((z[j] - mean) * rstd) : 0.0f;
      }
      s1 += t;
      s2 += u;
    }
    const float c1 = block_sum((float)s1, sm[0]) / (float)a.cols, c2 = block_sum((float)s2, sm[1]) / (float)a.cols;
    for (long long c = threadIdx.x * 8; c < a.cols; c += 2048) {
      const int nv = (int)min(8ll, a.cols - c);
      const bool drop = load_z<TX, TR, RES>(a, key, row, c, nv, z, m);
      load_param_some<TX>(a.weight, a.p_f32, c, nv, 1.0f, w);
      Vec8<TR> d;
      load_nv(d, reinterpret_cast<const TR*>(a.dy) + row * a.ld_dy + c, nv);
#pragma unroll
      for (int j = 0; j < 8; ++j) z[j] = rstd * (d.get(j) * w[j] - c1 - (z[j] - mean) * rstd * c2);
      if (RES && a.dresidual != nullptr) {
        d.set(z);
        d.store(reinterpret_cast<TR*>(a.dresidual) + row * a.cols + c, nv);
      }
      if (a.dx != nullptr) {
        if (drop) {
#pragma unroll
          for (int j = 0; j < 8; ++j) z[j] = m.kept(j, keep_limit(a.drop.tm1)) ? z[j] * a.drop.scale : 0.0f;
        }
        Vec8<TX> o;
        o.set(z);
        o.store(reinterpret_cast<TX*>(a.dx) + row * a.cols + c, nv);
      }
    }
  }
}

// partial[g][0 / 1][cols]: sums of dy xhat and of dy over the rows g, g + G, ...; a thread owns eight columns.  The wider the rows, the fewer partial
// sums there are (one from 2 million columns on), so 64 rows add up in fp32 and these sums in fp64.
template <class TX, class TR, int RES>
__global__ __launch_bounds__(256) void norm_wide_dw_kernel(NormArgs a) {
  DropKey key{};
  if (RES) key = drop_key(a.drop);
  const long long c = ((long long)blockIdx.x * 256 + threadIdx.x) * 8;
  if (c >= a.cols) return;
  const int nv = (int)min(8ll, a.cols - c);
  double dw64[8] = {}, db64[8] = {};
  float dw[8] = {}, db[8] = {}, z[8];
  const auto flush = [&] {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      dw64[j] += dw[j];
      db64[j] += db[j];
      dw[j] = db[j] = 0.0f;
    }
  };
  Keep8 m;
  int left = 64;
  for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
    if (left-- == 0) {
      flush();
      left = 63;
    }
    const float mean = a.mean[row], rstd = a.rstd[row];
    load_z<TX, TR, RES>(a, key, row, c, nv, z, m);
    Vec8<TR> d;
    load_nv(d, reinterpret_cast<const TR*>(a.dy) + row * a.ld_dy + c, nv);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      dw[j] = fmaf(d.get(j), (z[j] - mean) * rstd, dw[j]);
      db[j] += d.get(j);
    }
  }
  flush();
  float* p = a.workspace + (long long)blockIdx.y * 2 * a.cols + c;
  for (int j = 0; j < nv; ++j) {
    p[j] = (float)dw64[j];
    p[a.cols + j] = (float)db64[j];
  }
}

int norm_wide_parts(long long rows, long long cols) {
  const long long slabs = (cols + 2047) / 2048;                     // workgroups along the columns; fill ~1024 with rows
  long long g = (1024 + slabs - 1) / slabs;
  if (g > rows) g = rows;
  return (int)(g < 1 ? 1 : g);
}

template <class TX, class TR, int RES> static int wide_forward(const NormArgs& a, hipStream_t s) {
  const unsigned grid = grid_of(a.rows, 256);
  norm_wide_fwd_kernel<TX, TR, RES><<<grid, 256, 0, s>>>(a);
  return check_launch("norm_forward");
}
template <class TX, class TR, int RES> static int wide_backward(const NormArgs& a, hipStream_t s) {
  if (a.rows > 0 && (a.dx != nullptr || a.dresidual != nullptr)) {
    const unsigned grid = grid_of(a.rows, 256);
    norm_wide_dx_kernel<TX, TR, RES><<<grid, 256, 0, s>>>(a);
    if (check_launch("norm_backward")) return -1;
  }
  if (a.dweight != nullptr || a.dbias != nullptr) {
    const int parts = norm_wide_parts(a.rows, a.cols);
    norm_wide_dw_kernel<TX, TR, RES><<<dim3((unsigned)((a.cols + 2047) / 2048), parts), 256, 0, s>>>(a);
    if (check_launch("norm_backward")) return -1;
    return norm_finish(a, parts, s);
  }
  return 0;
}

int norm_wide_forward(const NormArgs& a, hipStream_t stream) { NORM_DISPATCH(wide_forward, a, stream); }
int norm_wide_backward(const NormArgs& a, hipStream_t stream) { NORM_DISPATCH(wide_backward, a, stream); }

}  // namespace lbm
