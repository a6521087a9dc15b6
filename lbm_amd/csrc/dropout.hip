// Dropout with a mask that is drawn where it is used and never stored: y = keep ? x * scale : 0.  The gradient is the same map of dy.
#include "train.hpp"

namespace lbm {

int make_drop(double p, uint64_t seed, const void* seed_ptr, uint64_t offset, DropArgs& d) {
  LBM_REQUIRE(p >= 0.0 && p <= 1.0, "dropout: p = %g is not a probability", p);
  LBM_REQUIRE(((uintptr_t)seed_ptr & 7) == 0, "dropout: the seed tensor must be 8-byte aligned");
  const uint64_t t = (uint64_t)__builtin_nearbyint(p * 4294967296.0);    // exact product, one rounding
  d.on = t != 0;
  d.tm1 = t == 0 ? 0u : (uint32_t)(t - 1);
  d.scale = t >= 4294967296ull ? 0.0f : (float)(4294967296.0 / (double)(4294967296ull - t));
  d.seed = seed;
  d.seed_ptr = reinterpret_cast<const uint64_t*>(seed_ptr);
  d.offset = offset;
  return 0;
}

// A thread takes one chunk of eight elements, which is one block of the generator, and ends (beyond 2^35 elements it strides, since a launch
// holds no more threads): bound by HBM (67108864 bf16 46 us, 5.8 TB/s;
// 150994944 bf16 99 us, 6.1; fp32 207 us, 5.8: its lanes lie 32 bytes apart).  A grid that strides over the chunks
// instead reached 4.4 - 5.0 TB/s; the ten rounds are hidden behind the memory (0, 7 or 10 of them: 345, 347, 342 us a GiB).
template <class T>
__global__ __launch_bounds__(256) void dropout_kernel(const T* x, T* y, long long n, DropArgs d) {
  const DropKey key = drop_key(d);
  const uint32_t limit = keep_limit(d.tm1);
  const long long chunks = (n + 7) >> 3, step = (long long)gridDim.x * 256;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < chunks; i += step) {
    const long long left = n - 8 * i;
    const int nv = left < 8 ? (int)left : 8;
    Vec8<T> v;
    if (nv == 8) v.load(x + 8 * i);
    else v.load_some(x + 8 * i, nv);
    if (d.on) {
      const Keep8 m = block_keep((uint64_t)i, key, d.tm1);
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = m.kept(j, limit) ? v.get(j) * d.scale : 0.0f;
      v.set(f);
    }
    v.store(y + 8 * i, nv);
  }
}

int dropout(const void* x, void* y, long long n, int type, const DropArgs& d, hipStream_t stream) {
  if (n == 0) return 0;
  ProfScope prof("dropout", stream, 3.0 * n, 2.0 * n * elem_size(type));
  const long long chunks = (n + 7) >> 3, want = (chunks + 255) / 256;
  const unsigned grid = grid_of(want, 256);
  switch (type) {
    case kF32: dropout_kernel<float><<<grid, 256, 0, stream>>>((const float*)x, (float*)y, n, d); break;
    case kF16: dropout_kernel<_Float16><<<grid, 256, 0, stream>>>((const _Float16*)x, (_Float16*)y, n, d); break;
    default: dropout_kernel<__bf16><<<grid, 256, 0, stream>>>((const __bf16*)x, (__bf16*)y, n, d); break;
  }
  return check_launch("dropout");
}

}  // namespace lbm
