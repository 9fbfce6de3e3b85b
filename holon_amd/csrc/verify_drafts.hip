// Drafted tokens judged against the target's probabilities, from given random numbers. Request b owns rows start[b] ..
// start[b + 1] - 1 of the logits; row i judges drafted[i], the last one has none behind it. With p = softmax(logits / T) and q the
// distribution that the draft came from (given, or certainty):
//
//   row i takes its draft x when accept[i] q(x) < p(x);   after the first that does not (or the last row) one token is drawn:
//   from max(p - q, 0), renormalised, where a draft was turned down, from p where none was judged,
//   the first x with sum_{y <= x} mass(y) > draw[b] * sum mass.
//
// So a token's law is p whatever q is: accept lies in [0, 1), where it is below p(x) / q(x) with that probability (1 at most), and never
// where p(x) = 0, at accept[i] = 0 and q(x) = 0 too: what a mask has set to -inf does not come out. T = 0 takes the largest logit for p.
// The draw compares a running sum over up to hundreds of thousands of masses with a given number: exponentials and sums are in 64 bits,
// where the order of a sum moves a border between two tokens by 1e-16 of the whole, not by more than a token's own mass as in 32.
//
// Two launches over pieces of 4,096 values: every row's largest value and sum of exponentials; the judgement and the walk through the
// one piece that the drawn number falls into, by a block a request. The masses of p are the pieces' sums, those of p without a certain
// draft too but for its own piece; where drafts came with probabilities, a launch between judges (every block for itself) and sums
// max(p - q, 0) of the rows whose draft was turned down. 151,936 tokens, 64 requests of four drafts: 45 us (177 MB of logits, 3.9 TB/s:
// memory, and beside it 64-bit arithmetic, 34 us by its count), 22 and 11; one request of three 4.4, 6.4 and 9.0, each a chain of loads.
// Without probabilities 44 and 16 (its launch between took 13 us more a call), 4.4 and 11.5.
// (The walk by the last block to leave its masses, which saves a launch, took the judgement's launch over 64 requests from 28 to 111 us:
// to see the others' masses across the XCDs each block writes back and drops what its L2 holds of the logits.)
#include "common.h"
#include "holon_hip.h"

namespace {

constexpr int PIECE = 4096, THREADS = 256, EACH = PIECE / THREADS, MOST = 64;   // MOST: rows a request may have
constexpr int NONE = 0x7fffffff;

struct RowPart {        // of one piece of one row
  double sum;           // of 2^((l - max) c), c = log2(e) / T
  float max;
  int at;               // the first place of `max`
};
struct Judged {         // of one request
  double inv_z;         // 1 / sum of the end row
  double heat;          // log2(e) / T; 0: T = 0, the token is known
  float max;            // of the end row
  int row, accepted, draft;   // the end row (-1: no rows), how many drafts were taken, the one that was not (-1: none was judged)
  int token;
};

// exp((l - max) / T) as 2^z, z = (l - max) c with c = log2(e) / T: 2^n times, on [-1/2, 1/2], the sum of (r ln 2)^k / k! up to
// k = 11, whose next term is at most 7e-15. Adding 1.5 2^52 rounds z to a whole number and leaves it in the low bits, from where it
// goes into the exponent: three additions where rounding, converting and scaling each take four times an addition's cycles.
// 1 at the largest value, also where that is infinite; nothing below 2^-1000 of it, and nothing for what is no number.
struct Weight {
  double c, max64, k[12];
  bool infinite;
  float max;
  // (The coefficients come from scalar registers: known to the compiler, each would be moved into the vector register that its
  // product adds to, two moves a product.)
  __device__ __forceinline__ Weight(float max_, double c_) : c(c_), max64(max_), infinite(fabsf(max_) == INFINITY), max(max_) {
    constexpr double L = 0.69314718055994530942;
    double term = 1.0;
#pragma unroll
    for (int i = 0; i < 12; ++i) {
      k[i] = term;
      term *= L / (i + 1);
      asm("" : "+s"(k[i]));
    }
    if (infinite) max64 = 0.0;
  }
  // What a row's value counts as: where the largest is infinite, 0 for those that are, and nothing for the others.
  __device__ __forceinline__ float value(float l) const { return !infinite ? l : l == max && max > 0.f ? 0.f : -INFINITY; }
  __device__ __forceinline__ double of_value(float l) const {
    constexpr double MAGIC = 6755399441055744.0;
    const double z = ((double)l - max64) * c, t = z + MAGIC, r = z - (t - MAGIC);      // (exactly 0 at the largest, however small T is)
    double p = k[11];
#pragma unroll
    for (int i = 10; i >= 0; --i) p = fma(p, r, k[i]);
    const uint64_t bits = __builtin_bit_cast(uint64_t, p);
    const uint32_t high = (uint32_t)(bits >> 32) + ((uint32_t)__builtin_bit_cast(uint64_t, t) << 20);
    return z >= -1000.0 ? __builtin_bit_cast(double, (uint64_t)high << 32 | (uint32_t)bits) : 0.0;
  }
  __device__ __forceinline__ double operator()(float l) const { return of_value(value(l)); }
  template <int N> __device__ __forceinline__ void prepare(float (&x)[N]) const {      // `value` of all, where it changes any
    if (__any(infinite)) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = value(x[i]);
    }
  }
};

// The values of piece `lo` that a thread takes: 4 * (tid + 256 j) .. + 3, j < 4, in 16-byte loads where rows allow it.
__device__ __forceinline__ void load_piece(const float* __restrict__ row, int lo, int vocab, bool wide, float fill, float (&x)[EACH]) {
  if (wide && lo + PIECE <= vocab) {
    float4 v[EACH / 4];
#pragma unroll
    for (int j = 0; j < EACH / 4; ++j) v[j] = *reinterpret_cast<const float4*>(row + lo + 4 * ((int)threadIdx.x + THREADS * j));
#pragma unroll
    for (int j = 0; j < EACH / 4; ++j) { x[4 * j] = v[j].x; x[4 * j + 1] = v[j].y; x[4 * j + 2] = v[j].z; x[4 * j + 3] = v[j].w; }
    return;
  }
#pragma unroll
  for (int j = 0; j < EACH / 4; ++j) {
    const int at = lo + 4 * ((int)threadIdx.x + THREADS * j);
    if (wide && at + 3 < vocab) {
      const float4 v = *reinterpret_cast<const float4*>(row + at);
      x[4 * j] = v.x; x[4 * j + 1] = v.y; x[4 * j + 2] = v.z; x[4 * j + 3] = v.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * j + e] = at + e < vocab ? row[at + e] : fill;
    }
  }
}
__device__ __forceinline__ int place_of(int lo, int i) { return lo + 4 * ((int)threadIdx.x + THREADS * (i / 4)) + i % 4; }

__device__ __forceinline__ double wave_sum64(double v) {
  v += lane_xor<32>(v);
  v += lane_xor<16>(v);
  v += lane_xor<8>(v);
  v += lane_xor<4>(v);
  v += lane_xor<2>(v);
  v += lane_xor<1>(v);
  return v;
}
__device__ __forceinline__ double block_sum64(double v, double* part) {      // every thread gets it; `part`: 4 values of LDS
  v = wave_sum64(v);
  if (threadIdx.x % WAVE == 0) part[threadIdx.x / WAVE] = v;
  __syncthreads();
  const double s = (part[0] + part[1]) + (part[2] + part[3]);
  __syncthreads();
  return s;
}

// The request that owns row i (-1: none): how many starts are at most i, by the lanes of a wave side by side.
__device__ __forceinline__ int owner_of(const int32_t* __restrict__ start, int requests, int i) {
  int before = 0;
  for (int at = 0; at <= requests; at += WAVE) {
    const int j = at + (int)(threadIdx.x % WAVE);
    before += __popcll(__ballot(j <= requests && start[min(j, requests)] <= i));
  }
  return before >= 1 && before <= requests ? before - 1 : -1;
}
// log2(e) / T; 0 says T = 0 (an infinite T: all the same but what is -inf).
__device__ __forceinline__ double heat_of(float t) { return t > 0.f ? fmax(1.4426950408889634074 / (double)t, 1e-300) : 0.0; }

__global__ void __launch_bounds__(THREADS) verify_rows_kernel(const float* __restrict__ logits, const int32_t* __restrict__ start,
                                                              const float* __restrict__ temperature, RowPart* __restrict__ parts,
                                                              int requests, int vocab, int wide) {
  __shared__ RowPart of_wave[THREADS / WAVE];
  const int piece = blockIdx.x, row = blockIdx.y, lo = piece * PIECE;
  float x[EACH];
  load_piece(logits + (int64_t)row * vocab, lo, vocab, wide, -INFINITY, x);
  const int b = owner_of(start, requests, row);
  if (b < 0) return;                                          // a row behind the last request's (the same for the whole block)
  const double c = heat_of(temperature[b]);
  // each wave by itself, under its own largest value: one barrier a block
  float top = x[0] > -INFINITY ? x[0] : -INFINITY;            // (what is no number is never larger)
#pragma unroll
  for (int i = 1; i < EACH; ++i) top = fmaxf(top, x[i]);
  top = wave_max(top);
  int at = NONE;
  double s = 0.0;
  if (c > 0.0) {
    const Weight weight(top, c);
    weight.prepare(x);
#pragma unroll
    for (int i = 0; i < EACH; ++i) s += weight.of_value(x[i]);
    s = wave_sum64(s);
  } else {                                                    // T = 0: where the largest stands first
#pragma unroll
    for (int i = EACH - 1; i >= 0; --i)
      if (x[i] == top && top > -INFINITY) at = place_of(lo, i);
#pragma unroll
    for (int o = WAVE / 2; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o, WAVE));
  }
  if (threadIdx.x % WAVE == 0) of_wave[threadIdx.x / WAVE] = RowPart{s, top, at};
  __syncthreads();
  if (threadIdx.x < WAVE) {                                   // the four waves' by lanes 0 .. 3, added in that order
    const RowPart mine = of_wave[threadIdx.x % (THREADS / WAVE)];
    const float most = lanes_max<THREADS / WAVE>(mine.max);
    double sum = c > 0.0 ? mine.sum * Weight(most, c)(mine.max) : 0.0;
    int first = mine.max == most ? mine.at : NONE;
    sum += lane_xor<1>(sum);
    sum += lane_xor<2>(sum);
    first = min(first, lane_xor<1>(first));
    first = min(first, lane_xor<2>(first));
    if (threadIdx.x == 0) parts[(int64_t)row * gridDim.x + piece] = RowPart{sum, most, first};
  }
}

// One wave: a row's largest value, its first place and its sum of weights from its pieces, added in piece order by lanes and
// then over the lanes: an order that the number of pieces alone decides.
__device__ __forceinline__ RowPart whole_row(const RowPart* __restrict__ parts, int pieces, double c) {
  const int lane = threadIdx.x % WAVE;
  float top = -INFINITY;
  int at = NONE;
  for (int i = lane; i < pieces; i += WAVE) {
    const RowPart p = parts[i];
    if (p.max > top || (p.max == top && p.at < at)) { top = p.max; at = p.at; }
  }
#pragma unroll
  for (int o = WAVE / 2; o > 0; o >>= 1) {
    const float t2 = __shfl_xor(top, o, WAVE);
    const int a2 = __shfl_xor(at, o, WAVE);
    if (t2 > top || (t2 == top && a2 < at)) { top = t2; at = a2; }
  }
  double s = 0.0;
  if (c > 0.0) {
    const Weight weight(top, c);
    for (int i = lane; i < pieces; i += WAVE) s += parts[i].sum * weight(parts[i].max);
  }
  return RowPart{wave_sum64(s), top, at};
}

// Running sums over a wave's lanes and a block's threads, each one's own among them; in an order that is the same for every call.
__device__ __forceinline__ double wave_upto64(double v) {
  const int lane = threadIdx.x % WAVE;
#pragma unroll
  for (int o = 1; o < WAVE; o *= 2) {
    const double before = __shfl_up(v, o, WAVE);
    if (lane >= o) v += before;
  }
  return v;
}
__device__ __forceinline__ double block_upto64(double v, double* part) {
  const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
  v = wave_upto64(v);
  if (lane == WAVE - 1) part[wave] = v;
  __syncthreads();
  double base = 0.0;
  for (int w = 0; w < wave; ++w) base += part[w];
  __syncthreads();
  return base + v;
}
__device__ __forceinline__ int block_min(int v, int* part) {
#pragma unroll
  for (int o = WAVE / 2; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, WAVE));
  if (threadIdx.x % WAVE == 0) part[threadIdx.x / WAVE] = v;
  __syncthreads();
  v = min(min(part[0], part[1]), min(part[2], part[3]));
  __syncthreads();
  return v;
}

// What a block judges by: the request's rows and all that was drafted for them.
struct Request {
  const float* logits;
  const int32_t* drafted;
  const float* draft_probs;    // nullable
  const float* accept;
  const float* temperature;
  const int32_t* start;
  const RowPart* parts;
  int rows, pieces, vocab, most;
};
// The judgement of request b, by every thread of a block.
__device__ __forceinline__ Judged judge(const Request& r, int b) {
  __shared__ RowPart whole[MOST];
  __shared__ int verdict[MOST];                               // 1: taken, 0: turned down, -1: nothing to judge
  const int wave = threadIdx.x / WAVE, lane = threadIdx.x % WAVE;
  const int first = max(r.start[b], 0), n = min(min(r.start[b + 1], r.rows) - first, r.most + 1);
  if (n <= 0) return Judged{0.0, 0.0, 0.f, -1, 0, -1, -1};
  const double c = heat_of(r.temperature[b]);
  for (int i = wave; i < n; i += THREADS / WAVE) {
    const int row = first + i, x = r.drafted[row];            // (what the judgement needs is asked for before the sums are added)
    const bool may = i + 1 < n && x >= 0 && x < r.vocab;
    const int64_t at = (int64_t)row * r.vocab + (may ? x : 0);
    const float lx = r.logits[at], qx = r.draft_probs != nullptr ? r.draft_probs[at] : 1.f, u = r.accept[row];
    const RowPart w = whole_row(r.parts + (int64_t)row * r.pieces, r.pieces, c);
    const bool good = c > 0.0 ? (double)u * (double)qx * w.sum < Weight(w.max, c)(lx) : x == (w.at == NONE ? 0 : w.at);
    if (lane == 0) {
      whole[i] = w;
      verdict[i] = may ? (good ? 1 : 0) : -1;
    }
  }
  __syncthreads();
  int end = 0;
  while (end < n - 1 && verdict[end] == 1) ++end;
  const RowPart w = whole[end];
  const int row = first + end;
  return Judged{w.sum > 0.0 ? 1.0 / w.sum : 0.0, c, w.max, row, end, verdict[end] == 0 ? r.drafted[row] : -1, w.at == NONE ? 0 : w.at};
}

// Where drafts came with probabilities: what max(p - q, 0) leaves of each piece of a row whose draft was turned down. (All else that is
// drawn from, the rows' own sums say.)
__global__ void __launch_bounds__(THREADS) verify_masses_kernel(Request r, Judged* __restrict__ judged, double* __restrict__ masses, int wide) {
  __shared__ double part[THREADS / WAVE];
  const int piece = blockIdx.x, b = blockIdx.y;
  const Judged j = judge(r, b);
  if (piece == 0 && threadIdx.x == 0) judged[b] = j;
  if (j.draft < 0 || j.heat == 0.0) return;
  float x[EACH], q[EACH];
  load_piece(r.logits + (int64_t)j.row * r.vocab, piece * PIECE, r.vocab, wide, -INFINITY, x);
  load_piece(r.draft_probs + (int64_t)j.row * r.vocab, piece * PIECE, r.vocab, wide, 0.f, q);
  const Weight weight(j.max, j.heat);
  weight.prepare(x);
  double left = 0.0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) left += fmax(weight.of_value(x[i]) * j.inv_z - (double)q[i], 0.0);
  left = block_sum64(left, part);
  if (threadIdx.x == 0) masses[(int64_t)b * r.pieces + piece] = left;
}

__global__ void __launch_bounds__(THREADS) verify_draw_kernel(Request r, const float* __restrict__ draw, const Judged* __restrict__ judged,
                                                              const double* __restrict__ masses, int32_t* __restrict__ tokens,
                                                              int32_t* __restrict__ accepted, int wide) {
  __shared__ double part[THREADS / WAVE];
  __shared__ int ints[THREADS / WAVE];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid % WAVE, pieces = r.pieces, vocab = r.vocab;
  const bool probs = r.draft_probs != nullptr;
  const double* mine = masses + (int64_t)b * pieces;
  const double early = probs ? mine[min(lane, pieces - 1)] : 0.0;      // (asked for with the judgement)
  const float u = draw[b];
  const Judged j = probs ? judged[b] : judge(r, b);
  int token = j.token;
  if (j.row >= 0 && j.heat > 0.0) {
    const Weight weight(j.max, j.heat);
    const float* row = r.logits + (int64_t)j.row * vocab;
    const RowPart* sums = r.parts + (int64_t)j.row * pieces;
    enum { FROM_P, BUT_DRAFT, LEFT };                        // what is drawn from: p, p without the draft that was certain, max(p - q, 0)
    int from = j.draft < 0 ? FROM_P : probs ? LEFT : BUT_DRAFT;
    // A certain draft's piece is summed without it: its weight taken off the piece's sum would leave rounding where nothing is.
    double without = 0.0;
    if (from == BUT_DRAFT) {
      const int lo = j.draft / PIECE * PIECE;
      float x[EACH];
      load_piece(row, lo, vocab, wide, -INFINITY, x);
      weight.prepare(x);
#pragma unroll
      for (int i = 0; i < EACH; ++i) without += place_of(lo, i) == j.draft ? 0.0 : weight.of_value(x[i]);
      without = block_sum64(without, part);
    }
    // Masses of 64 pieces, a lane's each: what is left over, or (not divided by the row's sum) what the rows' kernel summed.
    const auto mass = [&](int at) {
      const int i = at + lane;
      if (i >= pieces) return 0.0;
      if (from == LEFT) return at == 0 ? early : mine[i];
      if (from == BUT_DRAFT && i == j.draft / PIECE) return without;
      const RowPart p = sums[i];
      return p.sum * weight(p.max);
    };
    // Every wave finds the piece for itself, 64 pieces at a time: the one in which the running sum passes the target, or (a number
    // so near one that rounding passed the last border) the last one with any mass.
    double total = 0.0;
    for (;;) {
      for (int at = 0; at < pieces; at += WAVE) total += mass(at);
      total = wave_sum64(total);
      if (total > 0.0 || from == FROM_P) break;
      from = FROM_P;                                         // (q = p everywhere leaves nothing: then from p)
      total = 0.0;
    }
    const double target = (double)u * total;
    int heavy = NONE;
    double base = 0.0, carry = 0.0;
    for (int at = 0; at < pieces; at += WAVE) {
      const double m = mass(at), upto = carry + wave_upto64(m);
      const uint64_t over = __ballot(m > 0.0 && upto > target), some = __ballot(m > 0.0);
      if (over | some) {
        const int pick = over ? __ffsll((unsigned long long)over) - 1 : 63 - __clzll((long long)some);
        heavy = at + pick;
        base = __shfl(upto - m, pick, WAVE);
      }
      carry = __shfl(upto, WAVE - 1, WAVE);
      if (over) break;
    }
    token = 0;                                                // no token has any mass
    if (heavy != NONE) {
      const int lo = heavy * PIECE + tid * EACH;
      const float* qrow = r.draft_probs + (int64_t)j.row * vocab;
      float v[EACH], q[EACH];
      double m[EACH], s = 0.0;
      int last = -1;
#pragma unroll
      for (int i = 0; i < EACH; ++i) v[i] = lo + i < vocab ? row[lo + i] : -INFINITY;
#pragma unroll
      for (int i = 0; i < EACH; ++i) q[i] = from == LEFT && lo + i < vocab ? qrow[lo + i] : 0.f;
      weight.prepare(v);
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const int x = lo + i;
        double p = weight.of_value(v[i]);
        if (from == LEFT) p = fmax(p * j.inv_z - (double)q[i], 0.0);
        else if (from == BUT_DRAFT && x == j.draft) p = 0.0;
        m[i] = p;
        s += p;
        if (p > 0.0) last = x;
      }
      double sum = base + (block_upto64(s, part) - s);
      int found = NONE;
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        sum += m[i];
        if (m[i] > 0.0 && sum > target) found = min(found, lo + i);
      }
      found = block_min(found, ints);
      if (found == NONE) last = -block_min(-last, ints);
      token = found != NONE ? found : max(last, 0);
    }
  }
  for (int i = tid; i <= r.most; i += THREADS)
    tokens[(int64_t)b * (r.most + 1) + i] = j.row < 0 || i > j.accepted ? -1 : i == j.accepted ? token : r.drafted[j.row - j.accepted + i];
  if (tid == 0) accepted[b] = j.accepted;
}

}  // namespace

extern "C" int64_t holon_verify_drafts_room(int rows, int requests, int vocab) {
  const int64_t pieces = ((int64_t)vocab + PIECE - 1) / PIECE;
  return (rows * (int64_t)sizeof(RowPart) + requests * (int64_t)sizeof(double)) * pieces + requests * (int64_t)sizeof(Judged);
}

extern "C" int holon_verify_drafts(const float* logits, const int32_t* drafted, const float* draft_probs, const float* accept,
                                   const float* draw, const float* temperature, const int32_t* start, int32_t* tokens,
                                   int32_t* accepted, void* room, int rows, int requests, int vocab, int most, void* stream) {
  HOLON_CHECK(rows >= 0 && requests >= 0 && vocab > 0 && vocab <= PIECE * 65535, "verify_drafts: bad sizes");
  HOLON_CHECK(most >= 0 && most < MOST, "verify_drafts: %d drafted tokens a request (at most %d)", most, MOST - 1);
  HOLON_CHECK(rows <= 65535 && requests <= 65535, "verify_drafts: %d rows of %d requests (at most 65,535)", rows, requests);
  if (requests == 0) return 0;
  const int pieces = (vocab + PIECE - 1) / PIECE;
  RowPart* parts = (RowPart*)room;
  double* masses = (double*)(parts + (int64_t)rows * pieces);
  Judged* judged = (Judged*)(masses + (int64_t)requests * pieces);
  const bool wide = vocab % 4 == 0 && ((uintptr_t)logits | (uintptr_t)draft_probs) % 16 == 0;
  hipStream_t s = (hipStream_t)stream;
  if (rows > 0) {
    verify_rows_kernel<<<dim3(pieces, rows), THREADS, 0, s>>>(logits, start, temperature, parts, requests, vocab, wide);
    HOLON_LAUNCH_OK();
  }
  const Request r{logits, drafted, draft_probs, accept, temperature, start, parts, rows, pieces, vocab, most};
  if (draft_probs != nullptr) {
    verify_masses_kernel<<<dim3(pieces, requests), THREADS, 0, s>>>(r, judged, masses, wide);
    HOLON_LAUNCH_OK();
  }
  verify_draw_kernel<<<requests, THREADS, 0, s>>>(r, draw, judged, masses, tokens, accepted, wide);
  HOLON_LAUNCH_OK();
  return 0;
}
