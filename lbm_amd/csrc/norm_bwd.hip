// Gradients of layer normalisation in one sweep over memory: dy, x (and residual) in, dx (and dresidual) out, and the sums of dy xhat and
// of dy for weight and bias on the way.
//   z = x or residual + dropout(x) again, xhat = (z - mean) rstd, g = dy w, dz = rstd (g - mean(g) - xhat mean(g xhat))
// A team of threads (norm.hpp) holds a row in registers; a thread owns the same columns of every row that its team works on, so the sums
// over rows are private registers until the workgroup's teams are added up through LDS and written as one partial sum
// [2][cols] a workgroup.  norm_finish adds the partial sums in a fixed order: no atomics, the same bits every time.
#include <algorithm>

#include "norm.hpp"

namespace lbm {

// Where a workgroup's column sums go: its partial sum, or dweight / dbias themselves when there is only one workgroup.
template <class T> __device__ __forceinline__ void put_sum(void* p, long long c, float v) {
  if (p != nullptr) reinterpret_cast<T*>(p)[c] = (T)v;
}
template <class TX> __device__ __forceinline__ void put_part(const NormArgs& a, int which, long long c, float v) {
  if (gridDim.x > 1) a.workspace[((long long)blockIdx.x * 2 + which) * a.cols + c] = v;
  else if (a.p_f32) put_sum<float>(which == 0 ? a.dweight : a.dbias, c, v);
  else put_sum<TX>(which == 0 ? a.dweight : a.dbias, c, v);
}
template <class T> __device__ __forceinline__ void put_sums(void* p, long long c, const float (&v)[8], int nv) {
  if (p == nullptr) return;
  Vec8<T> o;
  o.set(v);
  o.store(reinterpret_cast<T*>(p) + c, nv);
}
template <class TX> __device__ __forceinline__ void put_parts(const NormArgs& a, int which, long long c, const float (&v)[8], int nv) {
  if (gridDim.x > 1) put_sums<float>(a.workspace + ((long long)blockIdx.x * 2 + which) * a.cols, c, v, nv);
  else if (a.p_f32) put_sums<float>(which == 0 ? a.dweight : a.dbias, c, v, nv);
  else put_sums<TX>(which == 0 ? a.dweight : a.dbias, c, v, nv);
}

template <class TX, class TR, int K> struct BwdRow {
  Vec8<TR> d[K];
  Vec8<TX> x[K];
  Vec8<TR> r[K];
  float mean, rstd;
};

// One row of a team: xhat and g = dy w from what was loaded, their two sums (s1 = sum g, s2 = sum g xhat), the columns' sums.
// w: this thread's weights, from LDS where K > 1 (their registers would cost a wave a SIMD; a fetch is two ds_read_b128 a chunk).
// gone: a row past the last one, of which nothing counts.
template <class TX, class TR, int RES, int K, bool BLK, LoadMode MODE>
__device__ __forceinline__ void bwd_row(const NormArgs& a, const DropKey& key, BwdRow<TX, TR, K>& in, const Span (&sp)[K], bool gone, long long row,
                                        int lanes, int tl, const float* w, float (&xh)[K][8], float (&g)[K][8], Keep8 (&m)[K],
                                        float (&dw)[K][8], float (&db)[K][8], float& s1, float& s2) {
  s1 = s2 = 0.0f;
  if (RES && a.drop.on) keep_row<K, BLK>(m, (uint64_t)(row * a.cols), key, a.drop.tm1, (int)a.cols, lanes, tl);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    in.x[k].template cut<MODE>(sp[k].cut);
    in.d[k].template cut<MODE>(gone ? 8 : sp[k].cut);
    if (RES) in.r[k].template cut<MODE>(sp[k].cut);
    if (RES && a.drop.on) {
      const uint32_t limit = keep_limit(a.drop.tm1);
#pragma unroll
      for (int j = 0; j < 8; ++j) xh[k][j] = join_one<RES>(in.x[k].get(j), in.r[k].get(j), m[k].kept(j, limit), a.drop.scale);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) xh[k][j] = join_one<RES>(in.x[k].get(j), RES ? in.r[k].get(j) : 0.0f, true, 1.0f);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) xh[k][j] = (xh[k][j] - in.mean) * in.rstd;
    if (gone || sp[k].cut != 0) {          // dy is zero there, but zero times an overflowed xhat is not
#pragma unroll
      for (int j = 0; j < 8; ++j) xh[k][j] = !gone && j < 8 - sp[k].cut ? xh[k][j] : 0.0f;
    }
    int at = (k * lanes + tl) * 8;
    if (K > 1) asm volatile("" : "+v"(at));  // fetch the weights again for every row: kept across rows they take 8 K registers
    const float* wk = K > 1 ? w + at : w;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float d = in.d[k].get(j);
      g[k][j] = d * wk[j];
      s1 += g[k][j];
      s2 = fmaf(g[k][j], xh[k][j], s2);
      dw[k][j] = fmaf(d, xh[k][j], dw[k][j]);
      db[k][j] += d;
    }
  }
}
template <class TX, class TR, int RES, int K>
__device__ __forceinline__ void bwd_put(const NormArgs& a, const Span (&sp)[K], long long at, int lanes, int tl, float c1, float c2, float rstd,
                                        const float (&xh)[K][8], const float (&g)[K][8], const Keep8 (&m)[K]) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (sp[k].cut == 8) continue;
    float dz[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) dz[j] = rstd * (fmaf(-xh[k][j], c2, g[k][j] - c1));
    const long long o = at + (k * lanes + tl) * 8;
    if (RES && a.dresidual != nullptr) {
      Vec8<TR> v;
      v.set(dz);
      v.store(reinterpret_cast<TR*>(a.dresidual) + o, 8 - sp[k].cut);
    }
    if (a.dx != nullptr) {
      if (RES && a.drop.on) {
        const uint32_t limit = keep_limit(a.drop.tm1);
#pragma unroll
        for (int j = 0; j < 8; ++j) dz[j] = m[k].kept(j, limit) ? dz[j] * a.drop.scale : 0.0f;
      }
      Vec8<TX> v;
      v.set(dz);
      v.store(reinterpret_cast<TX*>(a.dx) + o, 8 - sp[k].cut);
    }
  }
}

// Rows of lanes of a wave.  The next row's loads are issued when this row has become xhat and g, and pass behind its sums and stores.
// Eight waves a workgroup, one workgroup a CU: half the partial sums of four waves and two (150000 x 1024 join 315 -> 295 us, 16320 x 257 16.4 -> 15.1).
// Bound by HBM: 589824 x 256 bf16 173 us (5.2 TB/s), the join 277 us (5.5).  A grid that is no whole number a CU is not (640 workgroups of 256
// threads: the join 316 us, 512: 274), nor are contiguous rows a workgroup (191 us): neighbouring workgroups on neighbouring rows.
constexpr int kBwdThreads = 512, kBwdWaves = kBwdThreads / 64;
template <class TX, class TR, int RES, int K, LoadMode MODE>
__global__ __launch_bounds__(kBwdThreads) void norm_bwd_kernel(NormArgs a, int shift) {
  __shared__ __align__(16) float red[kBwdWaves * 512 * K];         // the weights (K > 1); at the end one column sum of every wave
  const int lanes = 1 << shift, tl = threadIdx.x & (lanes - 1), team = threadIdx.x >> shift, teams = kBwdThreads >> shift, cols = (int)a.cols;
  const float inv = 1.0f / (float)cols;
  DropKey key{};
  if (RES) key = drop_key(a.drop);
  Span sp[K];
  float w[8], dw[K][8] = {}, db[K][8] = {};
#pragma unroll
  for (int k = 0; k < K; ++k) {
    sp[k] = Span::of<MODE>((k * lanes + tl) * 8, cols, k == K - 1);
    if (K == 1 || (int)threadIdx.x < lanes) load_param<TX, MODE == kShort ? kShort : kPlain>(a.weight, a.p_f32, sp[k], 1.0f, w);
    if (K > 1 && (int)threadIdx.x < lanes) {
#pragma unroll
      for (int j = 0; j < 8; ++j) red[(k * lanes + tl) * 8 + j] = w[j];
    }
  }
  if (K > 1) __syncthreads();
  BwdRow<TX, TR, K> in;
  const auto load = [&](long long base) {                  // a team's row of the rows base .. base + teams - 1 (past the last: the last)
    const uint32_t r = min((long long)team, a.rows - base - 1);
    const TX* px = reinterpret_cast<const TX*>(a.x) + base * a.ld_x;
    const TR* pr = reinterpret_cast<const TR*>(a.residual) + base * a.ld_r;
    const TR* pd = reinterpret_cast<const TR*>(a.dy) + base * a.ld_dy;
    in.mean = a.mean[base + r];
    in.rstd = a.rstd[base + r];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      in.d[k].template load<MODE>(pd + row_at(r, (uint32_t)a.ld_dy, sp[k].at), 8 - sp[k].cut);
      in.x[k].template load<MODE>(px + row_at(r, (uint32_t)a.ld_x, sp[k].at), 8 - sp[k].cut);
      if (RES) in.r[k].template load<MODE>(pr + row_at(r, (uint32_t)a.ld_r, sp[k].at), 8 - sp[k].cut);
    }
  };
  const long long step = (long long)gridDim.x * teams;
  long long base = (long long)blockIdx.x * teams;
  if (base < a.rows) load(base);
  for (; base < a.rows; base += step) {
    const long long row = base + team;
    float xh[K][8], g[K][8], s1, s2;
    Keep8 m[K];
    const float rstd = in.rstd;
    bwd_row<TX, TR, RES, K, false, MODE>(a, key, in, sp, row >= a.rows, row, lanes, tl, K > 1 ? red : w, xh, g, m, dw, db, s1, s2);
    if (base + step < a.rows) load(base + step);
    const float c1 = lanes_sum(s1, shift) * inv, c2 = lanes_sum(s2, shift) * inv;
    if (row < a.rows) bwd_put<TX, TR, RES, K>(a, sp, row * a.cols, lanes, tl, c1, c2, rstd, xh, g, m);
  }
  if (a.dweight == nullptr && a.dbias == nullptr) return;
  // the teams of a wave, then the waves
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float(&acc)[K][8] = which == 0 ? dw : db;
    for (int s = lanes; s < 64; s <<= 1)
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[k][j] += __shfl_xor(acc[k][j], s);
    if (K > 1 || which == 1) __syncthreads();
    if ((int)(threadIdx.x & 63) < lanes) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) red[(threadIdx.x >> 6) * (512 * K) + (k * lanes + tl) * 8 + j] = acc[k][j];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < cols; c += kBwdThreads) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < kBwdWaves; ++i) s += red[i * (512 * K) + c];
      put_part<TX>(a, which, c, s);
    }
  }
}

// Rows of a workgroup.  AHEAD: the next row's loads pass behind this row's sums, as above, at the price of registers (512 threads at
// most); otherwise up to 1024 threads with 128 registers each, a row at a time.  18000 x 8192 bf16 165 - 184 us (4.8 - 5.4 TB/s), the join 270 - 285 us (5.2 - 5.5; a
// row at a time 303); 9000 x 16384 188 us (4.7: the partial sums are 7 % of the traffic), fp32 338 us (5.2), the join a row at a time 285 us (5.2), f16 beside an fp32
// residual 470 (5.0).  A few long rows are bound by one
// row's latency after the other (4096 x 2048: 20 us, eight rows a workgroup).
template <class TX, class TR, int RES, int K, bool AHEAD, LoadMode MODE>
__global__ __launch_bounds__(AHEAD ? 512 : 1024) void norm_bwd_block_kernel(NormArgs a) {
  extern __shared__ __align__(16) float wlds[];            // K * blockDim.x * 8 weights
  __shared__ float sums[2][16][2];
  const int lanes = blockDim.x, tl = threadIdx.x, cols = (int)a.cols;
  const float inv = 1.0f / (float)cols;
  DropKey key{};
  if (RES) key = drop_key(a.drop);
  Span sp[K];
  float dw[K][8] = {}, db[K][8] = {};
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float w[8];
    sp[k] = Span::of<MODE>((k * lanes + tl) * 8, cols, k == K - 1);
    load_param<TX, kPlain>(a.weight, a.p_f32, sp[k], 1.0f, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) wlds[(k * lanes + tl) * 8 + j] = w[j];      // read by this thread only
  }
  BwdRow<TX, TR, K> in;
  const auto load = [&](long long row) {
    const TX* px = reinterpret_cast<const TX*>(a.x) + row * a.ld_x;
    const TR* pr = reinterpret_cast<const TR*>(a.residual) + row * a.ld_r;
    const TR* pd = reinterpret_cast<const TR*>(a.dy) + row * a.ld_dy;
    in.mean = a.mean[row];
    in.rstd = a.rstd[row];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      in.d[k].template load<MODE>(pd + sp[k].at);
      in.x[k].template load<MODE>(px + sp[k].at);
      if (RES) in.r[k].template load<MODE>(pr + sp[k].at);
    }
  };
  if (AHEAD && blockIdx.x < a.rows) load(blockIdx.x);
  int half = 0;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    if (!AHEAD) load(row);
    float xh[K][8], g[K][8], s1, s2;
    Keep8 m[K];
    const float rstd = in.rstd;
    bwd_row<TX, TR, RES, K, true, MODE>(a, key, in, sp, false, row, lanes, tl, wlds, xh, g, m, dw, db, s1, s2);
    if (AHEAD && row + gridDim.x < a.rows) load(row + gridDim.x);
    // one barrier a row: the next row writes the other half, and the one after it finds every thread past this row's reads
    s1 = wave64_sum(s1);
    s2 = wave64_sum(s2);
    if ((tl & 63) == 0) {
      sums[half][tl >> 6][0] = s1;
      sums[half][tl >> 6][1] = s2;
    }
    __syncthreads();
    s1 = s2 = 0.0f;
    for (int i = 0; i < lanes >> 6; ++i) {
      s1 += sums[half][i][0];
      s2 += sums[half][i][1];
    }
    half ^= 1;
    bwd_put<TX, TR, RES, K>(a, sp, row * a.cols, lanes, tl, s1 * inv, s2 * inv, rstd, xh, g, m);
  }
  if (a.dweight == nullptr && a.dbias == nullptr) return;
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (sp[k].cut < 8) {
      put_parts<TX>(a, 0, (k * lanes + tl) * 8, dw[k], 8 - sp[k].cut);
      put_parts<TX>(a, 1, (k * lanes + tl) * 8, db[k], 8 - sp[k].cut);
    }
}

// dweight / dbias = the partial sums added up in a fixed order: 32 columns x 32 slices of the partial sums a workgroup.  4 - 5 us up to 8192 columns, 7 at
// 16384: latencies (8 dependent rounds of loads, a barrier, 32 reads), not bandwidth.
template <class T>
__global__ __launch_bounds__(1024) void norm_finish_kernel(const float* part, int parts, long long cols, T* dweight, T* dbias) {
  __shared__ float sm[32][33];
  const int tc = threadIdx.x & 31, tg = threadIdx.x >> 5;
  for (long long c0 = (long long)blockIdx.x * 32; c0 < 2 * cols; c0 += (long long)gridDim.x * 32) {      // over 2 cols: dweight, then dbias
    const long long c = c0 + tc;
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
    __syncthreads();
  }
}

int norm_finish(const NormArgs& a, int parts, hipStream_t s) {
  const unsigned grid = grid_of((2 * a.cols + 31) / 32, 1024);      // beyond 2^26 columns it strides
  if (a.p_f32) norm_finish_kernel<float><<<grid, 1024, 0, s>>>(a.workspace, parts, a.cols, (float*)a.dweight, (float*)a.dbias);
  else if (a.x_type == kF16) norm_finish_kernel<_Float16><<<grid, 1024, 0, s>>>(a.workspace, parts, a.cols, (_Float16*)a.dweight, (_Float16*)a.dbias);
  else norm_finish_kernel<__bf16><<<grid, 1024, 0, s>>>(a.workspace, parts, a.cols, (__bf16*)a.dweight, (__bf16*)a.dbias);
  return check_launch("norm_backward");
}

// The teams of the backward pass: more than 1536 columns belong to a workgroup (K = 4 in a wave leaves one wave a SIMD; between 1024 and
// 1536 a wave's 192 chunks waste less than a workgroup's 256: the join at 145348 x 1032 bf16 314 us, 504 in a workgroup).  Up to 8192 columns
// it has 512 threads at most, with registers for the loads ahead; beyond, K = 4 chunks a thread where they fit beside those (lean: half
// precision without a residual), else 1024 threads that load a row at a time.
static NormShape bwd_shape(long long cols, bool lean) {
  const int chunks = (int)((cols + 7) / 8);
  NormShape s = norm_shape(cols, 192);
  s.threads = kBwdThreads;
  if (chunks <= 192) return s;
  s = NormShape{chunks > 1024 && lean ? 4 : 2, 0, 0, true};
  s.threads = (chunks + 64 * s.k - 1) / (64 * s.k) * 64;
  return s;
}
// workgroups = partial sums: what is resident at once, a whole number a CU (the sums a workgroup keeps make the launch persistent)
static int norm_parts(long long rows, long long cols, bool lean) {
  const NormShape sh = bwd_shape(cols, lean);
  int per_cu = !sh.block ? 1 : sh.threads <= 128 ? 3 : sh.threads <= 256 ? 2 : 1;
  while (per_cu > 1 && rows < 8 * 256 * per_cu) --per_cu;      // a partial sum costs the traffic of two or three rows
  const long long g = (rows + sh.teams() - 1) / sh.teams();
  if (g <= (sh.block || sh.k > 1 ? 2 : 4)) return 1;
  // (a few rounds of one workgroup cost less than the second launch: 64 x 256 join 8.4 us and 8.7 with it, 2048 x 8 f32 7.1 and 9.3, 256 x 64 7.0 and 8.9, 16 x 512
  // 4.1 and 8.3, 16 x 1000 bf16 6.1 and 8.6, 2 x 8192 bf16 5.7 and 8.6; two rows of 16384 columns of an fp32 join 17.2 and 15.4)
  return (int)std::min(g, 256ll * per_cu);
}

uint64_t norm_workspace_bytes(long long rows, long long cols) {
  const int parts = cols > kNormRowMax ? norm_wide_parts(rows, cols) : std::max(norm_parts(rows, cols, false), norm_parts(rows, cols, true));
  return (uint64_t)parts * 2 * (uint64_t)cols * sizeof(float);
}

template <class TX, class TR, int RES, LoadMode MODE> static int backward_rows(const NormArgs& a, hipStream_t s) {
  constexpr bool lean = RES == 0 && sizeof(TX) == 2;
  const NormShape sh = bwd_shape(a.cols, lean);
  const int grid = norm_parts(a.rows, a.cols, lean);
  const size_t lds = (size_t)sh.threads * sh.k * 8 * sizeof(float);
  if (sh.block && sh.k == 4) norm_bwd_block_kernel<TX, TR, RES, lean ? 4 : 2, true, MODE><<<grid, sh.threads, lds, s>>>(a);
  else if (sh.block && sh.threads <= 512) norm_bwd_block_kernel<TX, TR, RES, 2, true, MODE><<<grid, sh.threads, lds, s>>>(a);
  else if (sh.block) norm_bwd_block_kernel<TX, TR, RES, 2, false, MODE><<<grid, sh.threads, lds, s>>>(a);
  else if (sh.k == 1) norm_bwd_kernel<TX, TR, RES, 1, MODE><<<grid, kBwdThreads, 0, s>>>(a, sh.shift);
  else if (sh.k == 2) norm_bwd_kernel<TX, TR, RES, 2, MODE><<<grid, kBwdThreads, 0, s>>>(a, sh.shift);
  else norm_bwd_kernel<TX, TR, RES, 3, MODE><<<grid, kBwdThreads, 0, s>>>(a, sh.shift);
  if (check_launch("norm_backward")) return -1;
  if (grid > 1 && (a.dweight != nullptr || a.dbias != nullptr)) return norm_finish(a, grid, s);
  return 0;
}

template <class TX, class TR, int RES> static int backward_short(const NormArgs& a, hipStream_t s) {
  const int grid = norm_parts(a.rows, a.cols, false);
  norm_bwd_kernel<TX, TR, RES, 1, kShort><<<grid, kBwdThreads, 0, s>>>(a, bwd_shape(a.cols, false).shift);
  if (check_launch("norm_backward")) return -1;
  if (grid > 1 && (a.dweight != nullptr || a.dbias != nullptr)) return norm_finish(a, grid, s);
  return 0;
}

template <class TX, class TR, int RES> static int backward(const NormArgs& a, hipStream_t s) {
  constexpr LoadMode odd = sizeof(TX) == 2 ? kOdd : kPlain;
  if (a.cols < 8) return backward_short<TX, TR, RES>(a, s);
  if (odd == kOdd && (odd_rows<TX>(a.x, a.ld_x) || odd_rows<TR>(a.dy, a.ld_dy) || (RES && odd_rows<TR>(a.residual, a.ld_r)))) return backward_rows<TX, TR, RES, odd>(a, s);
  return backward_rows<TX, TR, RES, kPlain>(a, s);
}

int norm_backward(const NormArgs& a, hipStream_t stream) {
  ProfScope prof("norm_backward", stream, 14.0 * a.rows * a.cols,
                 (double)a.rows * a.cols * (2.0 * elem_size(a.x_type) + elem_size(a.y_type) * (a.residual ? 3.0 : 1.0)));
  if (a.cols > kNormRowMax) return norm_wide_backward(a, stream);
  NORM_DISPATCH(backward, a, stream);
}

}  // namespace lbm
