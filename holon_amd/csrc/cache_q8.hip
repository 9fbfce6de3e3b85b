// The 8-bit paged cache: keys and values quantised as they are written, and read back (the format: cache_q8.h).
#include "cache_q8.h"
#include "holon_hip.h"

namespace {

constexpr int RUN = 16;      // tokens a block takes of one head: a run of 16 tokens of a page is 16 bytes of every dim's values

// The place of token t0 + i (i < 16) by lane i of each row of 16 lanes, as page * page_size + offset; -1: none (or no such token).
__device__ __forceinline__ int64_t place_of(const int32_t* __restrict__ page, const int32_t* __restrict__ off, int t, int tokens,
                                            int page_size, int num_pages) {
  if (t >= tokens) return -1;
  const int pg = page[t], at = off[t];
  return pg >= 0 && pg < num_pages && at >= 0 && at < page_size ? (int64_t)pg * page_size + at : -1;
}
// Whether 16 places are a run: one after the other from a border of 16 on (pages are multiples of 16, so they share one).
__device__ __forceinline__ bool is_run(const int64_t* places) {
  bool run = places[0] >= 0 && places[0] % RUN == 0;
#pragma unroll
  for (int i = 1; i < RUN; ++i) run &= places[i] == places[0] + i;
  return run;
}

template <typename T, int N>
__device__ __forceinline__ void load_values(const T* x, bool wide, float (&f)[N]) {
  if (wide) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(x + i);
        f[i] = v.x; f[i + 1] = v.y; f[i + 2] = v.z; f[i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const ushort4 v = *reinterpret_cast<const ushort4*>(x + i);
        f[i] = bf16_to_float(v.x); f[i + 1] = bf16_to_float(v.y); f[i + 2] = bf16_to_float(v.z); f[i + 3] = bf16_to_float(v.w);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = Elem<T>::load(x[i]);
  }
}

// A block takes 16 tokens of one head: 16 lanes a token, D / 16 values of its key and of its value a lane. Values go through LDS
// where their tokens are a run, so that 16 bytes of a dim are written at once; tokens anywhere else have theirs written one by one.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv_write_q8_kernel(const T* __restrict__ k, const T* __restrict__ v, int64_t stride, int wide,
                                                          uint8_t* __restrict__ pages, uint8_t* __restrict__ scales,
                                                          int64_t page_stride, int64_t scale_stride,
                                                          const int32_t* __restrict__ write_page,
                                                          const int32_t* __restrict__ write_off, int tokens, int kv_heads,
                                                          int page_size, int num_pages) {
  constexpr int E = D / 16;                                // values a lane
  __shared__ int64_t places[RUN];
  __shared__ __attribute__((aligned(16))) uint8_t turned[D][RUN];
  const int t0 = blockIdx.x * RUN, hk = blockIdx.y, i = threadIdx.x / 16, lane = threadIdx.x % 16, t = t0 + i;
  const int64_t place = place_of(write_page, write_off, t, tokens, page_size, num_pages);
  if (lane == 0) places[i] = place;
  float x[2][E];
  if (t < tokens) {
    const int64_t at = (int64_t)t * stride + (int64_t)hk * D + lane * E;
    load_values<T, E>(k + at, wide, x[0]);
    load_values<T, E>(v + at, wide, x[1]);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) x[0][e] = x[1][e] = 0.f;
  }
  uint32_t codes[2][E / 4], byte[2];
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    float most = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) most = fmaxf(most, q8_size(x[part][e]));
    byte[part] = q8_scale(lanes_max<16>(most));
    const float inverse = q8_inverse(byte[part]);
#pragma unroll
    for (int e = 0; e < E; e += 4)
      codes[part][e / 4] = q8_codes(x[part][e] * inverse, x[part][e + 1] * inverse, x[part][e + 2] * inverse, x[part][e + 3] * inverse);
  }
  __syncthreads();
  const bool run = is_run(places);
  const int64_t plane = (int64_t)page_size * D, page = place >= 0 ? place / page_size : 0;
  const int off = place >= 0 ? (int)(place % page_size) : 0;
  if (place >= 0) {
    uint32_t* to = reinterpret_cast<uint32_t*>(pages + page * page_stride + hk * plane + (int64_t)off * D + lane * E);
#pragma unroll
    for (int e = 0; e < E / 4; ++e) to[e] = codes[0][e];
    if (lane < 2) scales[page * scale_stride + ((int64_t)lane * kv_heads + hk) * page_size + off] = (uint8_t)(lane ? byte[1] : byte[0]);
  }
  if (run) {
#pragma unroll
    for (int e = 0; e < E; ++e) turned[lane * E + e][i] = (uint8_t)(codes[1][e / 4] >> (8 * (e % 4)));
    __syncthreads();
    uint8_t* to = pages + page * page_stride + (kv_heads + hk) * plane + places[0] % page_size;
    for (int d = threadIdx.x; d < D; d += 256)
      *reinterpret_cast<q8x4_t*>(to + (int64_t)d * page_size) = *reinterpret_cast<const q8x4_t*>(turned[d]);
  } else if (place >= 0) {
    uint8_t* to = pages + page * page_stride + (kv_heads + hk) * plane + off;
#pragma unroll
    for (int e = 0; e < E; ++e) to[(int64_t)(lane * E + e) * page_size] = (uint8_t)(codes[1][e / 4] >> (8 * (e % 4)));
  }
}

__device__ __forceinline__ void widen4(uint32_t w, float power, float (&f)[4]) {
  f[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0) * power;
  f[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * power;
  f[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * power;
  f[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * power;
}
template <typename T>
__device__ __forceinline__ void store4(T* to, const float (&f)[4]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(to) = float4{f[0], f[1], f[2], f[3]};
  } else {
    ushort4 w;
    w.x = float_to_bf16(f[0]); w.y = float_to_bf16(f[1]); w.z = float_to_bf16(f[2]); w.w = float_to_bf16(f[3]);
    *reinterpret_cast<ushort4*>(to) = w;
  }
}

// The same blocks the other way round: 16 lanes a token, D / 16 of its codes a lane.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv_read_q8_kernel(T* __restrict__ k, T* __restrict__ v, const uint8_t* __restrict__ pages,
                                                         const uint8_t* __restrict__ scales, int64_t page_stride,
                                                         int64_t scale_stride, const int32_t* __restrict__ read_page,
                                                         const int32_t* __restrict__ read_off, int tokens, int kv_heads,
                                                         int page_size, int num_pages) {
  constexpr int E = D / 16;
  __shared__ int64_t places[RUN];
  __shared__ __attribute__((aligned(16))) uint8_t turned[RUN][D + 16];
  const int t0 = blockIdx.x * RUN, hk = blockIdx.y, i = threadIdx.x / 16, lane = threadIdx.x % 16, t = t0 + i;
  const int64_t place = place_of(read_page, read_off, t, tokens, page_size, num_pages);
  if (lane == 0) places[i] = place;
  const int64_t plane = (int64_t)page_size * D, page = place >= 0 ? place / page_size : 0;
  const int off = place >= 0 ? (int)(place % page_size) : 0;
  const uint8_t* from = pages + page * page_stride + hk * plane;
  const uint8_t* powers = scales + page * scale_stride + (int64_t)hk * page_size + off;
  uint32_t codes[2][E / 4];
  uint32_t byte[2] = {powers[0], powers[(int64_t)kv_heads * page_size]};
#pragma unroll
  for (int e = 0; e < E / 4; ++e) codes[0][e] = *reinterpret_cast<const uint32_t*>(from + (int64_t)off * D + lane * E + 4 * e);
  from += kv_heads * plane;
  __syncthreads();
  if (is_run(places)) {
    for (int d = threadIdx.x; d < D; d += 256) {
      const q8x4_t w = *reinterpret_cast<const q8x4_t*>(from + (int64_t)d * page_size + places[0] % page_size);
#pragma unroll
      for (int r = 0; r < RUN; ++r) turned[r][d] = (uint8_t)(w[r / 4] >> (8 * (r % 4)));
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E / 4; ++e) codes[1][e] = *reinterpret_cast<const uint32_t*>(&turned[i][lane * E + 4 * e]);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t c = from[(int64_t)(lane * E + e) * page_size + off];
      codes[1][e / 4] = e % 4 ? codes[1][e / 4] | c << (8 * (e % 4)) : c;
    }
  }
  if (t >= tokens) return;
  const bool there = place >= 0;
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    T* to = (part ? v : k) + ((int64_t)t * kv_heads + hk) * D + lane * E;
    const float power = q8_power(byte[part]);
#pragma unroll
    for (int e = 0; e < E / 4; ++e) {
      float f[4] = {0.f, 0.f, 0.f, 0.f};
      if (there) widen4(codes[part][e], power, f);
      store4<T>(to + 4 * e, f);
    }
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
  const int size = dtype == HOLON_F32 ? 4 : 2;             // four values at once where every token's begin on a border of as many
  const int wide = ((uintptr_t)k | (uintptr_t)v | (uintptr_t)(stride * size)) % (4 * size) == 0;
#define CALL(T, D)                                                                                                              \
  kv_write_q8_kernel<T, D><<<dim3((tokens + RUN - 1) / RUN, kv_heads), 256, 0, (hipStream_t)stream>>>(                          \
      (const T*)k, (const T*)v, stride, wide, (uint8_t*)pages, (uint8_t*)scales, page_stride, scale_stride, write_page,         \
      write_off, tokens, kv_heads, page_size, num_pages)
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
  kv_read_q8_kernel<T, D><<<dim3((tokens + RUN - 1) / RUN, kv_heads), 256, 0, (hipStream_t)stream>>>(                           \
      (T*)k, (T*)v, (const uint8_t*)pages, (const uint8_t*)scales, page_stride, scale_stride, read_page, read_off, tokens,      \
      kv_heads, page_size, num_pages)
  FOR_TYPE_AND_SIZE(CALL);
#undef CALL
  HOLON_LAUNCH_OK();
  return 0;
}
