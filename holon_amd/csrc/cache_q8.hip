// The 8-bit paged cache: keys and values quantised as they are written, and read back (the format: cache_q8.h).
#include "cache_q8.h"
#include "holon_hip.h"

namespace {

template <typename T> __device__ __forceinline__ float as_float(T v) { return Elem<T>::load(v); }

// One wave a (token, head, keys or values).
template <typename T, int D>
__global__ void __launch_bounds__(128) kv_write_q8_kernel(const T* __restrict__ k, const T* __restrict__ v, int64_t stride,
                                                          uint8_t* __restrict__ pages, uint8_t* __restrict__ scales,
                                                          int64_t page_stride, int64_t scale_stride,
                                                          const int32_t* __restrict__ write_page,
                                                          const int32_t* __restrict__ write_off, int kv_heads, int page_size,
                                                          int num_pages) {
  constexpr int E = D / WAVE;
  const int t = blockIdx.x, hk = blockIdx.y, part = threadIdx.x / WAVE, lane = threadIdx.x % WAVE;
  const int pg = write_page[t], off = write_off[t];
  if (pg < 0 || pg >= num_pages || off < 0 || off >= page_size) return;
  const T* x = (part ? v : k) + (int64_t)t * stride + (int64_t)hk * D + lane * E;
  float f[E], most = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    f[i] = as_float<T>(x[i]);
    most = fmaxf(most, q8_size(f[i]));
  }
  const uint32_t byte = q8_scale(wave_max(most));
  const float inverse = q8_inverse(byte);
  uint8_t* plane = pages + pg * page_stride + ((int64_t)part * kv_heads + hk) * page_size * D;
  float g[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < E; ++i) g[i] = f[i] * inverse;
  const uint32_t w = q8_codes(g[0], g[1], g[2], g[3]);
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int d = lane * E + i;
    plane[part ? (int64_t)d * page_size + off : (int64_t)off * D + d] = (uint8_t)(w >> (8 * i));
  }
  if (lane == 0) scales[pg * scale_stride + ((int64_t)part * kv_heads + hk) * page_size + off] = (uint8_t)byte;
}

template <typename T, int D>
__global__ void __launch_bounds__(128) kv_read_q8_kernel(T* __restrict__ k, T* __restrict__ v, const uint8_t* __restrict__ pages,
                                                         const uint8_t* __restrict__ scales, int64_t page_stride,
                                                         int64_t scale_stride, const int32_t* __restrict__ read_page,
                                                         const int32_t* __restrict__ read_off, int kv_heads, int page_size,
                                                         int num_pages) {
  constexpr int E = D / WAVE;
  const int t = blockIdx.x, hk = blockIdx.y, part = threadIdx.x / WAVE, lane = threadIdx.x % WAVE;
  const int pg = read_page[t], off = read_off[t];
  T* y = (part ? v : k) + ((int64_t)t * kv_heads + hk) * D + lane * E;
  const bool there = pg >= 0 && pg < num_pages && off >= 0 && off < page_size;
  const uint8_t* plane = pages + (there ? pg : 0) * page_stride + ((int64_t)part * kv_heads + hk) * page_size * D;
  const int at = there ? off : 0;
  const float power = q8_power(scales[(there ? pg : 0) * scale_stride + ((int64_t)part * kv_heads + hk) * page_size + at]);
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int d = lane * E + i;
    const uint32_t code = plane[part ? (int64_t)d * page_size + at : (int64_t)at * D + d];
    const float f = __builtin_amdgcn_cvt_f32_fp8((int)code, 0) * power;
    y[i] = Elem<T>::store(there ? f : 0.f);
  }
}

}  // namespace

#define FOR_TYPE_AND_SIZE(CALL)                                             \
  do {                                                                      \
    if (dtype == HOLON_F32) {                                               \
      if (head_dim == 64) CALL(float, 64);                                  \
      else if (head_dim == 128) CALL(float, 128);                           \
      else CALL(float, 256);                                                \
    } else {                                                                \
      if (head_dim == 64) CALL(bf16_t, 64);                                 \
      else if (head_dim == 128) CALL(bf16_t, 128);                          \
      else CALL(bf16_t, 256);                                               \
    }                                                                       \
  } while (0)

static int q8_sizes(const char* what, int tokens, int kv_heads, int head_dim, int page_size, int num_pages, int64_t page_stride,
                    int64_t scale_stride, int dtype) {
  HOLON_CHECK(dtype == HOLON_F32 || dtype == HOLON_BF16, "%s: bad dtype", what);
  HOLON_CHECK(head_dim == 64 || head_dim == 128 || head_dim == 256, "%s: heads of %d (64, 128 and 256 are served)", what, head_dim);
  HOLON_CHECK(page_size > 0 && page_size % 16 == 0, "%s: pages of %d tokens (multiples of 16 are served)", what, page_size);
  HOLON_CHECK(tokens >= 0 && kv_heads > 0 && kv_heads <= 65535 && num_pages > 0, "%s: bad sizes", what);
  HOLON_CHECK(page_stride % 16 == 0 && scale_stride % 16 == 0 && page_stride >= 2ll * kv_heads * page_size * head_dim &&
                  scale_stride >= 2ll * kv_heads * page_size, "%s: pages lie on no borders of 16 bytes, or in one another", what);
  return 0;
}

extern "C" int holon_kv_write_q8(const void* k, const void* v, int64_t stride, void* pages, void* scales, int64_t page_stride,
                                 int64_t scale_stride, const int32_t* write_page, const int32_t* write_off, int tokens,
                                 int kv_heads, int head_dim, int page_size, int num_pages, int dtype, void* stream) {
  if (int rc = q8_sizes("kv_write_q8", tokens, kv_heads, head_dim, page_size, num_pages, page_stride, scale_stride, dtype)) return rc;
  HOLON_CHECK(stride >= (int64_t)kv_heads * head_dim, "kv_write_q8: tokens lie in one another");
  if (tokens == 0) return 0;
#define CALL(T, D)                                                                                                              \
  kv_write_q8_kernel<T, D><<<dim3(tokens, kv_heads), 128, 0, (hipStream_t)stream>>>(                                            \
      (const T*)k, (const T*)v, stride, (uint8_t*)pages, (uint8_t*)scales, page_stride, scale_stride, write_page, write_off,    \
      kv_heads, page_size, num_pages)
  FOR_TYPE_AND_SIZE(CALL);
#undef CALL
  HOLON_LAUNCH_OK();
  return 0;
}

extern "C" int holon_kv_read_q8(void* k, void* v, const void* pages, const void* scales, int64_t page_stride, int64_t scale_stride,
                                const int32_t* read_page, const int32_t* read_off, int tokens, int kv_heads, int head_dim,
                                int page_size, int num_pages, int dtype, void* stream) {
  if (int rc = q8_sizes("kv_read_q8", tokens, kv_heads, head_dim, page_size, num_pages, page_stride, scale_stride, dtype)) return rc;
  if (tokens == 0) return 0;
#define CALL(T, D)                                                                                                              \
  kv_read_q8_kernel<T, D><<<dim3(tokens, kv_heads), 128, 0, (hipStream_t)stream>>>(                                             \
      (T*)k, (T*)v, (const uint8_t*)pages, (const uint8_t*)scales, page_stride, scale_stride, read_page, read_off, kv_heads,    \
      page_size, num_pages)
  FOR_TYPE_AND_SIZE(CALL);
#undef CALL
  HOLON_LAUNCH_OK();
  return 0;
}
