// Layer normalisation with the row in registers: y = (z - mean) rstd w + b, z = x or residual + dropout(x).
// One sweep over memory: a team of threads (norm.hpp) loads its row, sums it, sums the deviations from that mean and their squares (the
// two-pass form; the deviations' own mean corrects the first one, norm.hpp) and writes y.  Bound by HBM: x (and residual) in, y out.
#include <algorithm>

#include "norm.hpp"

namespace lbm {

template <class TX, class TR, int K> struct FwdRow {
  Vec8<TX> x[K];
  Vec8<TR> r[K];
};

// z of a loaded row, its sum in s
template <class TX, class TR, int RES, int K, bool BLK, LoadMode MODE>
__device__ __forceinline__ float join_row(const NormArgs& a, const DropKey& key, FwdRow<TX, TR, K>& in, const Span (&sp)[K], long long row,
                                          int lanes, int tl, float (&z)[K][8]) {
  float s = 0.0f;
  Keep8 m[K];
  if (RES && a.drop.on) keep_row<K, BLK>(m, (uint64_t)(row * a.cols), key, a.drop.tm1, (int)a.cols, lanes, tl);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    in.x[k].template cut<MODE>(sp[k].cut);
    if (RES) in.r[k].template cut<MODE>(sp[k].cut);
    if (RES && a.drop.on) {
      const uint32_t limit = keep_limit(a.drop.tm1);
#pragma unroll
      for (int j = 0; j < 8; ++j) z[k][j] = join_one<RES>(in.x[k].get(j), in.r[k].get(j), m[k].kept(j, limit), a.drop.scale);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) z[k][j] = join_one<RES>(in.x[k].get(j), RES ? in.r[k].get(j) : 0.0f, true, 1.0f);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) s += z[k][j];              // what was cut is zero
  }
  return s;
}
// z -= mean; the sum of its squares and its own sum d over the elements that exist
template <int K> __device__ __forceinline__ float deviate(float (&z)[K][8], float mean, const Span (&sp)[K], float& d) {
  float s = d = 0.0f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int j = 0; j < 8; ++j) z[k][j] -= mean;
    if (sp[k].cut != 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j) z[k][j] = j < 8 - sp[k].cut ? z[k][j] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      s = fmaf(z[k][j], z[k][j], s);
      d += z[k][j];
    }
  }
  return s;
}
// dr = d rstd: (z - d) rstd in one instruction, off by e |d| rstd, and d is some e |mean| itself
template <class TR> __device__ __forceinline__ void put_y(TR* y, float (&z)[8], float dr, float rstd, const float (&w)[8], const float (&b)[8], int cut) {
#pragma unroll
  for (int j = 0; j < 8; ++j) z[j] = fmaf(fmaf(z[j], rstd, -dr), w[j], b[j]);
  Vec8<TR> o;
  o.set(z);
  o.store(y, 8 - cut);
}

// Rows of up to 2048 columns.  U rows a team are loaded before the first is used, and a workgroup ends after them: a grid in row order
// keeps the whole chip on neighbouring pages.  589824 x 256 bf16 107 us (5.6 TB/s), the join 158 us (5.7); 583657 x 257 139 us (4.3: the 33rd
// chunk of a row has a stripe of its own).  Beside HBM the vector instructions are next: 57 % of the issue slots at 256 columns.
template <class TX, class TR, int RES, int K, int U, LoadMode MODE>
__global__ __launch_bounds__(256) void norm_fwd_kernel(NormArgs a, int shift, long long first) {
  const int lanes = 1 << shift, tl = threadIdx.x & (lanes - 1), team = threadIdx.x >> shift, teams = 256 >> shift, cols = (int)a.cols;
  const float inv = 1.0f / (float)cols;
  DropKey key{};
  if (RES) key = drop_key(a.drop);
  Span sp[K];
#pragma unroll
  for (int k = 0; k < K; ++k) sp[k] = Span::of<MODE>((k * lanes + tl) * 8, cols, k == K - 1);
  const long long base = first + (long long)blockIdx.x * (teams * U);
  const int last = (int)min((long long)(teams * U), a.rows - base) - 1;          // of this workgroup's rows
  const TX* px = reinterpret_cast<const TX*>(a.x) + base * a.ld_x;
  const TR* pr = reinterpret_cast<const TR*>(a.residual) + base * a.ld_r;
  TR* py = reinterpret_cast<TR*>(a.y) + base * a.cols;
  FwdRow<TX, TR, K> in[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t r = min(u * teams + team, last);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      in[u].x[k].template load<MODE>(px + row_at(r, (uint32_t)a.ld_x, sp[k].at), 8 - sp[k].cut);
      if (RES) in[u].r[k].template load<MODE>(pr + row_at(r, (uint32_t)a.ld_r, sp[k].at), 8 - sp[k].cut);
    }
  }
  float w[K][8], b[K][8];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    load_param<TX, MODE == kShort ? kShort : kPlain>(a.weight, a.p_f32, sp[k], 1.0f, w[k]);
    load_param<TX, MODE == kShort ? kShort : kPlain>(a.bias, a.p_f32, sp[k], 0.0f, b[k]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int r = u * teams + team;
    float z[K][8];
    const float mean = product(lanes_sum(join_row<TX, TR, RES, K, false, MODE>(a, key, in[u], sp, base + r, lanes, tl, z), shift), inv);
    float d;
    float s = deviate<K>(z, mean, sp, d);
    lanes_sum2(s, d, shift);
    d = product(d, inv);
    const float rstd = rsqrt_newton(norm_variance(s * inv, d) + a.eps);
    if (r > last) continue;
    if (tl == 0 && a.mean != nullptr) {
      a.mean[base + r] = mean + d;
      a.rstd[base + r] = rstd;
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (sp[k].cut < 8) put_y<TR>(py + row_at(r, (uint32_t)cols, (k * lanes + tl) * 8), z[k], d * rstd, rstd, w[k], b[k], sp[k].cut);
  }
}

// Rows of a workgroup.  The next row's loads are issued when this row has become z, so they pass behind its two sums and its stores: with
// 512 or 1024 threads a row only one or two rows are on a CU, and without that its memory was idle half of the time (8192 x 8192 bf16
// 74 us, now 50: 5.4 TB/s; 9000 x 16384 114 us, 5.2).
template <class TX, class TR, int RES, int K, LoadMode MODE>
__global__ __launch_bounds__(1024) void norm_fwd_block_kernel(NormArgs a) {
  __shared__ float sm[16], sm2[16][2];
  const int lanes = blockDim.x, tl = threadIdx.x, cols = (int)a.cols;
  const float inv = 1.0f / (float)cols;
  DropKey key{};
  if (RES) key = drop_key(a.drop);
  Span sp[K];
#pragma unroll
  for (int k = 0; k < K; ++k) sp[k] = Span::of<MODE>((k * lanes + tl) * 8, cols, k == K - 1);
  FwdRow<TX, TR, K> in;
  const auto load = [&](long long row) {
    const TX* px = reinterpret_cast<const TX*>(a.x) + row * a.ld_x;
    const TR* pr = reinterpret_cast<const TR*>(a.residual) + row * a.ld_r;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      in.x[k].template load<MODE>(px + sp[k].at);
      if (RES) in.r[k].template load<MODE>(pr + sp[k].at);
    }
  };
  float w[K][8], b[K][8];
  load(blockIdx.x);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    load_param<TX, kPlain>(a.weight, a.p_f32, sp[k], 1.0f, w[k]);
    load_param<TX, kPlain>(a.bias, a.p_f32, sp[k], 0.0f, b[k]);
  }
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float z[K][8];
    float s = join_row<TX, TR, RES, K, true, MODE>(a, key, in, sp, row, lanes, tl, z), d;
    if (row + gridDim.x < a.rows) load(row + gridDim.x);
    const float mean = product(block_sum(s, sm), inv);
    s = deviate<K>(z, mean, sp, d);
    block_sum2(s, d, sm2);
    d = product(d, inv);
    const float rstd = rsqrt_newton(norm_variance(s * inv, d) + a.eps);
    if (tl == 0 && a.mean != nullptr) {
      a.mean[row] = mean + d;
      a.rstd[row] = rstd;
    }
    TR* py = reinterpret_cast<TR*>(a.y) + row * a.cols;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (sp[k].cut < 8) put_y<TR>(py + (k * lanes + tl) * 8, z[k], d * rstd, rstd, w[k], b[k], sp[k].cut);
  }
}

// Rows in flight a team when that still makes 2048 workgroups, else one:
//   layer_norm   four, with two or three chunks a lane two: 65536 x 256 f16 14.8 us with four, 16.1 with one (9216 x 256: 5.7 and 4.4); 65536 x 1000 bf16
//                52.8 us with two, 56.6 with one (8192 x 1000: the same)
//   the join     two where its rows are no multiple of eight, whose masks wait for other lanes: 400000 x 249 bf16 139 us with two, 152 with one; other rows
//                one, which leaves more waves: 131072 x 256 bf16 37.4 us with one, 40.3 with two, 2000000 x 64 f16 137 and 147, fp32 residuals the same
constexpr long long kManyGroups = 2048;
// Chunks that a wave may hold: the join's four a lane leave two waves a SIMD (93750 x 1600 bf16: 218 us, 181 in a workgroup), three do not
// (97656 x 1536: 166 us, 178 in a workgroup; f16 beside an fp32 residual 261 and 284).
template <int RES> constexpr int wave_chunks() { return RES ? 192 : 256; }
template <class TX, class TR, int RES, int K, int U, LoadMode MODE> static int wave_forward(const NormArgs& a, const NormShape& sh, hipStream_t s) {
  const long long per = (long long)sh.teams() * U, most = grid_most(256) * per;
  for (long long first = 0; first < a.rows; first += most) {       // more than one launch: rows of fewer than eight columns, 2^32 and more of them
    const long long rows = std::min(most, a.rows - first);
    norm_fwd_kernel<TX, TR, RES, K, U, MODE><<<(unsigned)((rows + per - 1) / per), 256, 0, s>>>(a, sh.shift, first);
    if (check_launch("norm_forward")) return -1;
  }
  return 0;
}
template <class TX, class TR, int RES, LoadMode MODE> static int forward_rows(const NormArgs& a, hipStream_t s) {
  const NormShape sh = norm_shape(a.cols, wave_chunks<RES>());
  if (sh.block) {
    const long long most = 256 * (1024 / sh.threads);      // what is resident at once (16 waves a CU), a whole number a CU
    norm_fwd_block_kernel<TX, TR, RES, 2, MODE><<<(unsigned)(a.rows < most ? a.rows : most), sh.threads, 0, s>>>(a);
    return check_launch("norm_forward");
  }
  constexpr int U1 = RES ? 2 : 4, U2 = RES ? 1 : 2;
  if constexpr (RES == 0)
    if (sh.k == 4) return wave_forward<TX, TR, RES, 4, 1, MODE>(a, sh, s);
  const bool many = a.rows >= (long long)sh.teams() * (sh.k == 1 ? U1 : U2) * kManyGroups && (RES == 0 || (a.cols & 7) != 0);
  if (sh.k == 1) return many ? wave_forward<TX, TR, RES, 1, U1, MODE>(a, sh, s) : wave_forward<TX, TR, RES, 1, 1, MODE>(a, sh, s);
  if constexpr (RES == 0 || MODE != kOdd)      // the join's two chunks a lane are always loaded plainly (below)
    if (sh.k == 2) return many ? wave_forward<TX, TR, RES, 2, U2, MODE>(a, sh, s) : wave_forward<TX, TR, RES, 2, 1, MODE>(a, sh, s);
  return many ? wave_forward<TX, TR, RES, 3, U2, MODE>(a, sh, s) : wave_forward<TX, TR, RES, 3, 1, MODE>(a, sh, s);
}
template <class TX, class TR, int RES> static int forward(const NormArgs& a, hipStream_t s) {
  constexpr LoadMode odd = sizeof(TX) == 2 ? kOdd : kPlain;
  if (a.cols < 8) return wave_forward<TX, TR, RES, 1, 1, kShort>(a, norm_shape(a.cols, 1), s);
  // (the join's two chunks a lane are the exception: 146914 x 1021 bf16 194 us with plain loads, 208 dword by dword; 190000 x 785 224 and 247; beside an
  // fp32 residual 264 and 275 at 160000 x 901, the same at 100000 x 1021)
  const NormShape sh = norm_shape(a.cols, wave_chunks<RES>());
  if (odd == kOdd && (odd_rows<TX>(a.x, a.ld_x) || (RES && odd_rows<TR>(a.residual, a.ld_r))) && !(RES && !sh.block && sh.k == 2)) return forward_rows<TX, TR, RES, odd>(a, s);
  return forward_rows<TX, TR, RES, kPlain>(a, s);
}

int norm_forward(const NormArgs& a, hipStream_t stream) {
  if (a.rows == 0) return 0;
  ProfScope prof("norm_forward", stream, 8.0 * a.rows * a.cols,
                 (double)a.rows * a.cols * (elem_size(a.x_type) + elem_size(a.y_type) * (a.residual ? 2.0 : 1.0)));
  if (a.cols > kNormRowMax) return norm_wide_forward(a, stream);
  NORM_DISPATCH(forward, a, stream);
}

}  // namespace lbm
