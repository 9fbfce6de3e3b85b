// The 8-bit paged cache: keys and values quantised as they are written, and read back (the format: cache_q8.h).
#include "cache_q8.h"
#include "holon_hip.h"

namespace {

constexpr int RUN = 16;      // tokens a block takes of one head: a run of 16 tokens of a page is 16 bytes of every dim's values

// The place of a token; page -1: none, or no such token.
struct Place {
  int page, off;
};
__device__ __forceinline__ Place place_of(const int32_t* __restrict__ page, const int32_t* __restrict__ off, int t, int tokens,
                                          int page_size, int num_pages) {
  if (t >= tokens) return Place{-1, 0};
  const int pg = page[t], at = off[t];
  return pg >= 0 && pg < num_pages && at >= 0 && at < page_size ? Place{pg, at} : Place{-1, 0};
}
// Sixteen tokens in two stretches at most, each of neighbours within 16 bytes of every dim's values: tokens 0 .. first - 1, and from
// there to count - 1; no token behind those has a place. A portion of a sequence is that wherever it begins (16 tokens from an odd
// place on lie on both sides of one border), and so are most ends of one sequence and beginnings of the next. `any` is false of others.
struct Stretches {
  bool any;
  int first, count;
  // By every wave for itself, from the places in LDS.
  __device__ __forceinline__ explicit Stretches(const Place* places) {
    const int lane = threadIdx.x % RUN;
    const Place mine = places[lane], before = places[max(lane - 1, 0)];
    const bool goes_on = mine.page == before.page && mine.off == before.off + 1 && mine.off % RUN != 0;
    const uint32_t there = (uint32_t)__ballot(mine.page >= 0) & 0xffffu, breaks = (uint32_t)__ballot(lane > 0 && !goes_on) & there;
    any = (there & (there + 1)) == 0 && (breaks & (breaks - 1)) == 0;
    count = __popc(there);
    first = breaks ? __ffs(breaks) - 1 : count;
  }
};

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

// Bytes lo .. hi - 1 of 16, in the widest pieces that lie on borders of their own width.
__device__ __forceinline__ void store_bytes(uint8_t* to, const uint8_t* from, int lo, int hi) {
  if (hi - lo == RUN) {
    *reinterpret_cast<q8x4_t*>(to) = *reinterpret_cast<const q8x4_t*>(from);
    return;
  }
  while (lo < hi) {
    if (lo % 8 == 0 && lo + 8 <= hi) {
      *reinterpret_cast<uint64_t*>(to + lo) = *reinterpret_cast<const uint64_t*>(from + lo);
      lo += 8;
    } else if (lo % 4 == 0 && lo + 4 <= hi) {
      *reinterpret_cast<uint32_t*>(to + lo) = *reinterpret_cast<const uint32_t*>(from + lo);
      lo += 4;
    } else if (lo % 2 == 0 && lo + 2 <= hi) {
      *reinterpret_cast<uint16_t*>(to + lo) = *reinterpret_cast<const uint16_t*>(from + lo);
      lo += 2;
    } else {
      to[lo] = from[lo];
      lo += 1;
    }
  }
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

// Where a block's 16 tokens go.
struct Target {
  uint8_t* pages;
  uint8_t* scales;
  int64_t page_stride, scale_stride;
  const int32_t* page;         // [tokens]
  const int32_t* off;
  int tokens, kv_heads, page_size, num_pages;
};

// A block's 16 tokens of head hk into the cache: thread 16 i + lane has values D / 16 lane .. of token t0 + i, x[0] of its key and
// x[1] of its value.
template <int D>
__device__ __forceinline__ void write_block(const Target& w, int hk, const Place& place, Place* places, const float (&x)[2][D / 16]) {
  constexpr int E = D / 16;
  __shared__ __attribute__((aligned(16))) uint8_t turned[2][D][RUN];
  const int i = threadIdx.x / 16, lane = threadIdx.x % 16;
  uint8_t* const pages = w.pages;
  const int64_t page_stride = w.page_stride, scale_stride = w.scale_stride;
  const int kv_heads = w.kv_heads, page_size = w.page_size;
  if (lane == 0) places[i] = place;
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
  const Stretches two(places);
  const int64_t plane = (int64_t)page_size * D;
  if (place.page >= 0) {
    uint32_t* to = reinterpret_cast<uint32_t*>(pages + place.page * page_stride + hk * plane + (int64_t)place.off * D + lane * E);
#pragma unroll
    for (int e = 0; e < E / 4; ++e) to[e] = codes[0][e];
    if (lane < 2) w.scales[place.page * scale_stride + ((int64_t)lane * kv_heads + hk) * page_size + place.off] = (uint8_t)(lane ? byte[1] : byte[0]);
  }
  if (two.any) {
    if (place.page >= 0) {
#pragma unroll
      for (int e = 0; e < E; ++e) turned[i >= two.first][lane * E + e][place.off % RUN] = (uint8_t)(codes[1][e / 4] >> (8 * (e % 4)));
    }
    __syncthreads();
    for (int at = threadIdx.x; at < 2 * D; at += 256) {
      const int x = at / D, d = at % D, from = x ? two.first : 0, n = (x ? two.count : two.first) - from;
      if (n <= 0) break;
      const Place begin = places[from];
      const int lo = begin.off % RUN;
      store_bytes(pages + begin.page * page_stride + (kv_heads + hk) * plane + (int64_t)d * page_size + begin.off - lo, turned[x][d], lo, lo + n);
    }
  } else if (place.page >= 0) {
    uint8_t* to = pages + place.page * page_stride + (kv_heads + hk) * plane + place.off;
#pragma unroll
    for (int e = 0; e < E; ++e) to[(int64_t)(lane * E + e) * page_size] = (uint8_t)(codes[1][e / 4] >> (8 * (e % 4)));
  }
}

// A block takes 16 tokens of one head: 16 lanes a token, D / 16 values of its key and of its value a lane. Values go through LDS
// where their tokens lie in two stretches, so that what a stretch has of a dim's 16 bytes is written at once; tokens anywhere else
// have theirs written one by one. Memory bounds it: 8 heads of 128 in bfloat16, over inputs that change from call to call 4,096 tokens
// from a page's begin on 11.6 us a call, 16,384 35, 32,768 63 (202 MB, 3.2 TB/s). Over the same again and again, which the Infinity
// Cache holds: 4,096 tokens (25 MB) from a page's begin on 9.0, from its sixth place on 10.6, anywhere 27; 32,768 tokens 46, 54 and 169. With
// one stretch alone, a byte at a time from the sixth place on, the second of these took 14.9 and 87. Below some 1,000 tokens the host's 8 us.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv_write_q8_kernel(const T* __restrict__ k, const T* __restrict__ v, int64_t stride, int wide, Target w) {
  constexpr int E = D / 16;
  __shared__ Place places[RUN];
  const int hk = blockIdx.y, lane = threadIdx.x % 16, t = blockIdx.x * RUN + threadIdx.x / 16;
  const Place place = place_of(w.page, w.off, t, w.tokens, w.page_size, w.num_pages);
  float x[2][E];
  if (t < w.tokens) {
    const int64_t at = (int64_t)t * stride + (int64_t)hk * D + lane * E;
    load_values<T, E>(k + at, wide, x[0]);
    load_values<T, E>(v + at, wide, x[1]);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) x[0][e] = x[1][e] = 0.f;
  }
  write_block<D>(w, hk, place, places, x);
}

// The merged projection's heads: queries and keys normed and turned, queries to q_out, keys and values into the cache. A block takes
// 16 tokens of one kv head, or of one query head; a value's partner in the rotation is eight lanes away.
// 32 heads over 8 of 128 in bfloat16: 8 tokens 4.7 us (a chain of loads: position, angles; place, stores), 64 5.6, 2,048 15.3 (46 MB, 3.0
// TB/s), 8,192 50 (189 MB, 3.8); into the 16-bit cache, by blocks of a token each, which read angles and places once, 3.4, 3.8, 12.1 and 40.
template <typename T, int D>
__global__ void __launch_bounds__(256) qk_norm_rope_write_q8_kernel(const T* __restrict__ qkv, T* __restrict__ q_out, int heads,
                                                                    const T* __restrict__ q_weight, const T* __restrict__ k_weight,
                                                                    int wide_weights, float eps, const float* __restrict__ table,
                                                                    int max_positions, const int32_t* __restrict__ positions, Target w) {
  constexpr int E = D / 16;
  __shared__ Place places[RUN];
  const int lane = threadIdx.x % 16, t = blockIdx.x * RUN + threadIdx.x / 16, row = min(t, w.tokens - 1);
  const bool is_q = (int)blockIdx.y >= w.kv_heads;
  const int head = is_q ? blockIdx.y - w.kv_heads : blockIdx.y;
  // all that a block reads is asked for before anything waits, the longest chain first
  const int pos = table != nullptr ? min(max(positions[row], 0), max_positions - 1) : 0;
  Place place = {-1, 0};
  if (!is_q) place = place_of(w.page, w.off, t, w.tokens, w.page_size, w.num_pages);
  const T* src = qkv + (int64_t)row * (heads + 2 * w.kv_heads) * D + lane * E;
  float x[2][E], weight[E], co[E], si[E];
  load_values<T, E>(src + (int64_t)(is_q ? head : heads + head) * D, true, x[0]);
  if (!is_q) load_values<T, E>(src + (int64_t)(heads + w.kv_heads + head) * D, true, x[1]);
  const bool norm = q_weight != nullptr;
  if (norm) load_values<T, E>((is_q ? q_weight : k_weight) + lane * E, wide_weights, weight);
  if (table != nullptr) {
    const float* cs = table + (int64_t)pos * D + lane % 8 * E;
    load_values<float, E>(cs, true, co);
    load_values<float, E>(cs + D / 2, true, si);
  }
  if (norm) {
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) sum += x[0][e] * x[0][e];
    const float inv = 1.0f / sqrtf(lanes_sum<16>(sum) / (float)D + eps);
#pragma unroll
    for (int e = 0; e < E; ++e) x[0][e] = Elem<T>::round((x[0][e] * inv) * weight[e]);
  }
  if (table != nullptr) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float other = lane_xor<8>(x[0][e]);
      x[0][e] = Elem<T>::round(lane < 8 ? x[0][e] * co[e] - other * si[e] : x[0][e] * co[e] + other * si[e]);
    }
  }
  if (!is_q) {
    write_block<D>(w, head, place, places, x);
  } else if (t < w.tokens) {
    T* to = q_out + ((int64_t)t * heads + head) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      const float four[4] = {x[0][e], x[0][e + 1], x[0][e + 2], x[0][e + 3]};
      store4<T>(to + e, four);
    }
  }
}

__device__ __forceinline__ void widen4(uint32_t w, float power, float (&f)[4]) {
  f[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0) * power;
  f[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * power;
  f[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * power;
  f[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * power;
}
// The same blocks the other way round: 16 lanes a token, D / 16 of its codes a lane. Two thirds of what it moves are the values it
// writes: over inputs that change from call to call 32,768 tokens of 8 heads of 128 into bfloat16 (202 MB) 46 us, into 32 bits (336 MB) 86 (4.4
// and 3.9 TB/s); over the same again and again 36 us from a page's begin on, 40 from its sixth place on, 84 anywhere, into 32 bits 92, 97, 147.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv_read_q8_kernel(T* __restrict__ k, T* __restrict__ v, const uint8_t* __restrict__ pages,
                                                         const uint8_t* __restrict__ scales, int64_t page_stride,
                                                         int64_t scale_stride, const int32_t* __restrict__ read_page,
                                                         const int32_t* __restrict__ read_off, int tokens, int kv_heads,
                                                         int page_size, int num_pages) {
  constexpr int E = D / 16;
  __shared__ Place places[RUN];
  __shared__ __attribute__((aligned(16))) uint8_t turned[2][RUN][D + 16];
  const int t0 = blockIdx.x * RUN, hk = blockIdx.y, i = threadIdx.x / 16, lane = threadIdx.x % 16, t = t0 + i;
  const Place place = place_of(read_page, read_off, t, tokens, page_size, num_pages);
  if (lane == 0) places[i] = place;
  const bool there = place.page >= 0;
  const int64_t plane = (int64_t)page_size * D, page = there ? place.page : 0;
  const int off = place.off;
  const uint8_t* from = pages + page * page_stride + hk * plane;
  const uint8_t* powers = scales + page * scale_stride + (int64_t)hk * page_size + off;
  uint32_t codes[2][E / 4];
  uint32_t byte[2] = {powers[0], powers[(int64_t)kv_heads * page_size]};
#pragma unroll
  for (int e = 0; e < E / 4; ++e) codes[0][e] = *reinterpret_cast<const uint32_t*>(from + (int64_t)off * D + lane * E + 4 * e);
  from += kv_heads * plane;
  __syncthreads();
  const Stretches two(places);
  if (two.any) {
    for (int at = threadIdx.x; at < 2 * D; at += 256) {    // (all 16 bytes of a dim, also where the stretch has some of them alone)
      const int x = at / D, d = at % D, start = x ? two.first : 0;
      if ((x ? two.count : two.first) <= start) break;
      const Place begin = places[start];
      const q8x4_t w = *reinterpret_cast<const q8x4_t*>(pages + begin.page * page_stride + (kv_heads + hk) * plane + (int64_t)d * page_size +
                                                        begin.off / RUN * RUN);
#pragma unroll
      for (int r = 0; r < RUN; ++r) turned[x][r][d] = (uint8_t)(w[r / 4] >> (8 * (r % 4)));
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E / 4; ++e) codes[1][e] = *reinterpret_cast<const uint32_t*>(&turned[i >= two.first][off % RUN][lane * E + 4 * e]);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t c = from[(int64_t)(lane * E + e) * page_size + off];
      codes[1][e / 4] = e % 4 ? codes[1][e / 4] | c << (8 * (e % 4)) : c;
    }
  }
  if (t >= tokens) return;
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
  const Target to{(uint8_t*)pages, (uint8_t*)scales, page_stride, scale_stride, write_page, write_off, tokens, kv_heads, page_size, num_pages};
#define CALL(T, D)                                                                                                              \
  kv_write_q8_kernel<T, D><<<dim3((tokens + RUN - 1) / RUN, kv_heads), 256, 0, (hipStream_t)stream>>>((const T*)k, (const T*)v, stride, wide, to)
  FOR_TYPE_AND_SIZE(CALL);
#undef CALL
  HOLON_LAUNCH_OK();
  return 0;
}

extern "C" int holon_qk_norm_rope_write_q8(const void* qkv, void* q_out, int tokens, int heads, int kv_heads, int head_dim, const void* q_weight,
                                           const void* k_weight, float eps, const float* table, int max_positions, const int32_t* positions,
                                           void* pages, void* scales, int64_t page_stride, int64_t scale_stride, const int32_t* write_page,
                                           const int32_t* write_off, int page_size, int num_pages, int dtype, void* stream) {
  if (int rc = q8_sizes("qk_norm_rope_write_q8", tokens, kv_heads, head_dim, page_size, num_pages, page_stride, scale_stride, dtype)) return rc;
  HOLON_CHECK(heads > 0 && heads <= 65535 - kv_heads, "qk_norm_rope_write_q8: %d heads", heads);
  HOLON_CHECK((q_weight == nullptr) == (k_weight == nullptr), "qk_norm_rope_write_q8: q and k norm weights must both be given or both be absent");
  HOLON_CHECK(table == nullptr || (positions != nullptr && max_positions > 0), "qk_norm_rope_write_q8: a rotation needs positions");
  HOLON_CHECK(((uintptr_t)qkv | (uintptr_t)table) % 16 == 0, "qk_norm_rope_write_q8: tensors have to lie on borders of 16 bytes");
  if (tokens == 0) return 0;
  const int wide = ((uintptr_t)q_weight | (uintptr_t)k_weight) % (dtype == HOLON_F32 ? 16 : 8) == 0;
  const Target to{(uint8_t*)pages, (uint8_t*)scales, page_stride, scale_stride, write_page, write_off, tokens, kv_heads, page_size, num_pages};
#define CALL(T, D)                                                                                                              \
  qk_norm_rope_write_q8_kernel<T, D><<<dim3((tokens + RUN - 1) / RUN, kv_heads + heads), 256, 0, (hipStream_t)stream>>>(        \
      (const T*)qkv, (T*)q_out, heads, (const T*)q_weight, (const T*)k_weight, wide, eps, table, max_positions, positions, to)
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
