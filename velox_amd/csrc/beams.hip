// Several continuations of one request (beams) for gfx950: which of them go on, and what they held moving with them.
//
// beam_select.  Beam w of a request stands at scores[w]; a continuation by token v is worth
//     value(w, v) = scores[w] + (logits[w, v] - max_w - log sum_u exp(logits[w, u] - max_w)),
// and the `keep` most valuable of all beams and tokens are wanted, best first, ties to the lowest (w, v).  Within a beam the order is the
// logits' own, so a row's best `keep` hold all that can be wanted of it; what decides between rows is the log-sum, in which a rounding to 32
// bits would change the order of near ones: sums and values are held in 64 bits.  One kernel reads the logits once, a piece of a row per
// workgroup, and leaves each piece's maximum, sum of exponentials and best `keep` in order; a second, one workgroup per request, joins them.
//
// A piece's best `keep`.  Each of a workgroup's four waves keeps a list of what may be wanted of the values it has seen.  It has two bounds: one that
// `keep` values of its own reach, the least of the maxima of as many groups of lanes, which a value must exceed to join the list (an
// equal one comes behind those that set the bound), and the least of the four waves' bounds for a quarter of `keep`, which it must reach.  Joining is soon the
// exception; a list that is full is cut to its best `keep`.  The waves read what bounds the others have published and wait for one
// another behind the first round alone.
//
// What bounds it, measured on MI355X: 512 rows of 152,064 tokens (64 requests of 8 beams, 311 MB) take 85 to 88 us a call, 3.6 TB/s; traced, where kernels are slower, 95 us
// (median of 30 calls, the least 88) and 7.6 for joining.  Variants of it were timed untraced, this kernel 83 us then: the same from the
// second-level cache alone 72 us, without the exponentials 34; from memory without them 60: vector instructions, 28 a logit, of which the exponential in 64
// bits is 16, and a stream that reaches 5.4 TB/s overlap by half.  (In 32 bits it would be 63 us, and the sums 1e-7 off where 6e-11 settles the order of near
// ones.)  Medians of traced calls, both kernels: 64 rows of 152,064 22.6 + 6.2 us, 168 of 32,003 18.8 + 11.4, 4 of 151,936 8.2 + 7.0: of these, launches, the first round, in
// which much joins the lists, and the lists' joining are most.
//
// reorder_states: row slots[b, j, p] of every tensor becomes what row slots[b, parents[b, j], p] was.  A thread owns a column of the rows of one
// request: it has read all that move before it writes any, and nobody else reads or writes that column, so the rows change places
// in the memory they are in.
#include "common.h"

// ---- selection ------------------------------------------------------------------------------------------------------------
constexpr int THREADS = 256;
constexpr int MOST_KEPT = 64;

// e^x for -693 <= x <= 693 in 64 bits, to 6e-11 of it: x log2(e) = k + f with |f| <= 1/2, and the polynomial of degree 7 that takes 2^f's values at
// the Chebyshev points of that range.  (Adding 1.5 2^52 leaves k in the sum's low bits; it goes into the exponent.)
__device__ __forceinline__ double exp_in_range(double x) {
  constexpr double LOG2_E = 1.4426950408889634074, ROUNDS = 6755399441055744.0;
  const double shifted = fma(x, LOG2_E, ROUNDS), f = fma(x, LOG2_E, -(shifted - ROUNDS));
  double e = 1.5303699001378845e-05;
  e = fma(e, f, 0.00015469729140704658);
  e = fma(e, f, 0.0013333478480888061);
  e = fma(e, f, 0.0096180256135980358);
  e = fma(e, f, 0.055504109063177154);
  e = fma(e, f, 0.24022651213495422);
  e = fma(e, f, 0.69314718055683411);
  e = fma(e, f, 0.99999999995956224);
  typedef uint32_t halves_t __attribute__((ext_vector_type(2)));
  halves_t bits = __builtin_bit_cast(halves_t, e);
  bits[1] += __builtin_bit_cast(halves_t, shifted)[0] << 20;
  return __builtin_bit_cast(double, bits);
}
// What is far below counts as nothing beside 1.  A wave's terms may exceed what they are relative to by e^ABOVE before that is moved; a term further
// below it than BELOW counts as one that far; sums further apart than APART are not added.  (All within what exp_in_range takes, with what
// 32 bits' rounding of the bounds adds below COARSE.  From there on numbers are 64 and more apart, and only the greatest themselves count.)
constexpr float ABOVE = 600.f, BELOW = 640.f, COARSE = 1073741824.f;
constexpr double APART = 690.0;
// a sum of exponentials relative to `from`, relative to `to` >= from
__device__ __forceinline__ double moved_sum(double sum, float from, float to) {
  const double down = (double)to - (double)from;
  return from == to ? sum : down < APART ? sum * exp_in_range(-down) : 0.0;
}

__device__ __forceinline__ uint32_t ordered_bits(float v) {  // compares like the number
  const uint32_t b = __float_as_uint(v);
  return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t o) { return __uint_as_float((o & 0x80000000u) != 0 ? o ^ 0x80000000u : ~o); }

__device__ __forceinline__ float just_below(float v) {  // -inf: -inf
  return v == 0.f ? -1.401298464e-45f : v > -INFINITY ? from_ordered(ordered_bits(v) - 1) : v;
}

// The operation over the lanes of a row of 16, on every one of them.
template <typename Op> __device__ __forceinline__ float over_row(float v, Op op) {
#define VELOX_WITH(CONTROL) v = op(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CONTROL, 0xf, 0xf, true)))
  VELOX_WITH(0xB1);   // the neighbour,
  VELOX_WITH(0x4E);   // the other two of four,
  VELOX_WITH(0x141);  // the other four of eight,
  VELOX_WITH(0x140);  // the other eight
#undef VELOX_WITH
  return v;
}
template <typename Op> __device__ __forceinline__ float over_wave(float v, Op op) {
  v = over_row(v, op);
  auto at = [&](int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane)); };
  return op(op(at(0), at(16)), op(at(32), at(48)));
}

// The same for 64 bits (any type of eight bytes).
template <typename V, typename Op> __device__ __forceinline__ V over_row_64(V v, Op op) {
  typedef int halves_t __attribute__((ext_vector_type(2)));
#define VELOX_WITH(CONTROL)                                                              \
  {                                                                                      \
    halves_t x = __builtin_bit_cast(halves_t, v);                                        \
    x[0] = __builtin_amdgcn_update_dpp(0, x[0], CONTROL, 0xf, 0xf, true);                \
    x[1] = __builtin_amdgcn_update_dpp(0, x[1], CONTROL, 0xf, 0xf, true);                \
    v = op(v, __builtin_bit_cast(V, x));                                                 \
  }
  VELOX_WITH(0xB1)
  VELOX_WITH(0x4E)
  VELOX_WITH(0x141)
  VELOX_WITH(0x140)
#undef VELOX_WITH
  return v;
}
template <typename V, typename Op> __device__ __forceinline__ V over_wave_64(V v, Op op) {
  typedef int halves_t __attribute__((ext_vector_type(2)));
  v = over_row_64(v, op);
  const halves_t x = __builtin_bit_cast(halves_t, v);
  auto at = [&](int lane) { return __builtin_bit_cast(V, halves_t{__builtin_amdgcn_readlane(x[0], lane), __builtin_amdgcn_readlane(x[1], lane)}); };
  return op(op(at(0), at(16)), op(at(32), at(48)));
}
struct Sum64 { __device__ __forceinline__ double operator()(double a, double b) const { return a + b; } };

struct PieceSum { double sum; float top; int unused; };  // sum of exp(logit - top); top: a number near the greatest logit
struct Candidate { float logit; int token; };            // token < 0: none

constexpr int WAVES = THREADS / 64;
constexpr int WAVE_LEFT = 512;  // a wave's list

// Grid (pieces, rows); a piece is `span` tokens, a multiple of four, the row's last one may have fewer.  sums: [row][piece]; candidates:
// [row][piece][keep], best first.  A round is UNITS loads of four tokens by every thread, the next one's in flight while one is worked.
template <int UNITS>
__global__ void __launch_bounds__(THREADS) beam_pieces_kernel(const float* __restrict__ logits, const float* __restrict__ scores, int vocab, int span, int keep, int pieces,
                                                              PieceSum* __restrict__ sums, Candidate* __restrict__ candidates) {
  constexpr int UNIT = 4 * THREADS, ROUND = UNITS * UNIT, PER_ROUND = 4 * UNITS;
  __shared__ __attribute__((aligned(16))) uint64_t left[WAVES * WAVE_LEFT];
  __shared__ double wave_sums[WAVES];
  __shared__ float wave_refs[WAVES], wave_bounds[WAVES], wave_tops[WAVES];
  __shared__ __attribute__((aligned(16))) float quarter_bounds[WAVES];
  __shared__ int num_left[WAVES], reaches[2][WAVES];

  const int row = blockIdx.y, piece = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Candidate* const out = candidates + ((size_t)row * pieces + piece) * keep;
  if (!(scores[row] > -INFINITY)) {  // a beam that is not there: its continuations are all alike, the first tokens come first
    for (int r = tid; r < keep; r += THREADS) out[r] = Candidate{-INFINITY, piece == 0 && r < vocab ? r : -1};
    if (tid == 0) sums[(size_t)row * pieces + piece] = PieceSum{0.0, -INFINITY, 0};
    return;
  }
  // (a row begins wherever the one before ends: loads of four numbers at any multiple of four bytes.  Which thread adds up which tokens
  // must not hang on that, or equal rows would differ in their sums' last bits)
  typedef float loose4_t __attribute__((ext_vector_type(4), aligned(4)));
  const int base = piece * span, here = min(span, vocab - base);  // the piece's first token, its tokens
  const float* const first = logits + (size_t)row * vocab + base;
  auto load = [&](float (&v)[PER_ROUND], int round) {
#pragma unroll
    for (int q = 0; q < UNITS; ++q) {
      const int start = round * ROUND + q * UNIT, place = start + 4 * tid;
      if (start + UNIT <= here) {  // (the same for every thread)
        const loose4_t x = *reinterpret_cast<const loose4_t*>(first + place);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * q + j] = x[j];
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * q + j] = place + j < here ? first[place + j] : -INFINITY;
      }
    }
  };
  auto key_of = [&](float value, int place) -> uint64_t {  // (a zero has one form)
    return (uint64_t)ordered_bits(value + 0.f) << 32 | (uint32_t)~place;
  };
  auto greatest = [](float a, float b) { return fmaxf(a, b); };
  auto least = [](float a, float b) { return fminf(a, b); };

  uint64_t* const list = left + wave * WAVE_LEFT;
  int count = 0;
  float mine = -INFINITY;          // the greatest that this lane has seen
  float bound = -INFINITY;         // at least `keep` values of the rounds before are not below it
  float ref = -INFINITY;           // what the sum's terms are relative to: any number that they do not exceed beyond 64 bits' range
  double sum = 0.0;
  auto cut = [&]() {  // the list's best `keep`
    uint64_t k[WAVE_LEFT / 64], limit = 0;
#pragma unroll
    for (int a = 0; a < WAVE_LEFT / 64; ++a) k[a] = 64 * a + lane < count ? list[64 * a + lane] : 0;
    for (int bit = 63; bit >= 0; --bit) {
      const uint64_t trial = limit | 1ull << bit;
      int reach = 0;
#pragma unroll
      for (int a = 0; a < WAVE_LEFT / 64; ++a) reach += __popcll(__ballot(k[a] >= trial));
      if (reach >= keep) limit = trial;
    }
    count = 0;
#pragma unroll
    for (int a = 0; a < WAVE_LEFT / 64; ++a) {
      const uint64_t lanes = __ballot(k[a] >= limit);
      if (k[a] >= limit) list[count + __builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, 0))] = k[a];
      count += __popcll(lanes);
    }
    return from_ordered((uint32_t)(limit >> 32));
  };
  float next_bound = -INFINITY;
  auto take = [&](bool wanted, float value, int place) {
    const uint64_t lanes = __ballot(wanted);
    if (lanes == 0) return;
    const int more = __popcll(lanes);
    if (count + more > WAVE_LEFT) next_bound = fmaxf(next_bound, cut());
    if (wanted) list[count + __builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, 0))] = key_of(value, place);
    count += more;
  };
  auto work = [&](const float (&v)[PER_ROUND], int round) {
    float most = -INFINITY;
#pragma unroll
    for (int e = 0; e < PER_ROUND; ++e) most = fmaxf(most, v[e]);  // (what is no number is left out)
    mine = fmaxf(mine, most);
    auto with_lanes = [&](float part, int groups_from) {  // the least maximum of 64, 32, 16, 8 or 4 groups of lanes, at least as many as asked for
      if (groups_from <= 32) part = fmaxf(part, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(part), 0xB1, 0xf, 0xf, true)));
      if (groups_from <= 16) part = fmaxf(part, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(part), 0x4E, 0xf, 0xf, true)));
      if (groups_from <= 8) part = fmaxf(part, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(part), 0x141, 0xf, 0xf, true)));
      if (groups_from <= 4) part = fmaxf(part, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(part), 0x140, 0xf, 0xf, true)));
      return over_wave(part, least);
    };
    next_bound = fmaxf(next_bound, with_lanes(mine, keep));
    const float quarter = with_lanes(mine, (keep + 3) / 4);
    volatile float* const published = quarter_bounds;
    if (round == 0) {
      if (lane == 0) published[wave] = quarter;
      __syncthreads();
    }
    const float joint = fminf(fminf(published[0], published[1]), fminf(published[2], published[3]));
    if (round > 0 && lane == 0) published[wave] = quarter;
    const float above = fmaxf(round == 0 ? just_below(next_bound) : bound, just_below(joint));
    const int at = round * ROUND + 4 * tid;
    if (__ballot(most > above) != 0) {
#pragma unroll
      for (int e = 0; e < PER_ROUND; ++e) take(v[e] > above, v[e], at + (e >> 2) * UNIT + (e & 3));
    }
    if (round == 0 && wave == 0) {  // with fewer numbers than `keep` the first of the others fill up: they are among the first `keep` tokens
#pragma unroll
      for (int e = 0; e < 4; ++e) take(!(v[e] > -INFINITY) && 4 * tid + e < min(keep, here), -INFINITY, 4 * tid + e);
    }
    bound = next_bound;
    if (__ballot(most - ref > (fabsf(ref) < COARSE ? ABOVE : 0.f)) != 0) {  // the first numbers, or far beyond all before
      const float now = over_wave(most, greatest);
      sum = moved_sum(sum, ref, now);
      ref = now;
    }
    if (!(fabsf(ref) < COARSE)) {
#pragma unroll
      for (int e = 0; e < PER_ROUND; ++e) sum += v[e] == ref && ref > -INFINITY ? 1.0 : 0.0;
    } else {
      const double from = (double)ref;
      const float floor = ref - BELOW;
      double second = 0.0;  // (what is no number counts as far below)
#pragma unroll
      for (int e = 0; e < PER_ROUND; e += 2) {
        sum += exp_in_range((double)fmaxf(floor, v[e]) - from);
        second += exp_in_range((double)fmaxf(floor, v[e + 1]) - from);
      }
      sum += second;
    }
  };
  {
    float a[PER_ROUND], b[PER_ROUND];
    const int rounds = (here + ROUND - 1) / ROUND;
    load(a, 0);
    for (int round = 0; round < rounds; round += 2) {
      load(b, round + 1);  // (beyond the piece: nothing is loaded)
      work(a, round);
      if (round + 1 >= rounds) break;
      load(a, round + 2);
      work(b, round + 1);
    }
  }

  // The waves' sums, and of their lists what reaches the greatest of their bounds.
  sum = over_wave_64(sum, Sum64());
  mine = over_wave(mine, greatest);
  if (lane == 0) {
    wave_tops[wave] = mine;
    wave_sums[wave] = sum;
    wave_refs[wave] = ref;
    wave_bounds[wave] = bound;
  }
  __syncthreads();
  float limit = -INFINITY, joint = INFINITY, top = -INFINITY, greatest_seen = -INFINITY;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    limit = fmaxf(limit, wave_bounds[w]);
    joint = fminf(joint, quarter_bounds[w]);
    top = fmaxf(top, wave_refs[w]);
    greatest_seen = fmaxf(greatest_seen, wave_tops[w]);
  }
  limit = fmaxf(limit, joint);
  // That may be several times `keep`: a higher limit that `keep` or hardly more reach, by halving what lies between.
  uint64_t k[WAVE_LEFT / 64];
#pragma unroll
  for (int a = 0; a < WAVE_LEFT / 64; ++a) k[a] = 64 * a + lane < count ? list[64 * a + lane] : 0;
  int turn = 0;
  auto reach_of = [&](uint32_t trial) {
    int own = 0;
#pragma unroll
    for (int a = 0; a < WAVE_LEFT / 64; ++a) own += __popcll(__ballot((uint32_t)(k[a] >> 32) >= trial));
    turn ^= 1;
    if (lane == 0) reaches[turn][wave] = own;
    __syncthreads();
    return reaches[turn][0] + reaches[turn][1] + reaches[turn][2] + reaches[turn][3];
  };
  uint32_t lo = ordered_bits(limit + 0.f), hi = ordered_bits(greatest_seen) + 1;
  for (int have = reach_of(lo); have > 2 * keep + 32 && hi - lo > 1;) {
    const uint32_t trial = lo + (hi - lo) / 2;
    const int reach = reach_of(trial);
    if (reach >= keep) {
      lo = trial;
      have = reach;
    } else {
      hi = trial;
    }
  }
  count = 0;
#pragma unroll
  for (int a = 0; a < WAVE_LEFT / 64; ++a) {
    const bool stays = (uint32_t)(k[a] >> 32) >= lo;
    const uint64_t lanes = __ballot(stays);
    if (stays) list[count + __builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, 0))] = k[a];
    count += __popcll(lanes);
  }
  if (lane == 0) num_left[wave] = count;
  __syncthreads();
  // four threads to a value, each with one wave's list of the others
  static_assert(WAVES == 4, "a list for each of the four");
  const int counts[WAVES] = {num_left[0], num_left[1], num_left[2], num_left[3]};
  const int total = counts[0] + counts[1] + counts[2] + counts[3];
  const uint64_t* const others = left + (tid & 3) * WAVE_LEFT;
  const int num_others = (tid & 3) == 0 ? counts[0] : (tid & 3) == 1 ? counts[1] : (tid & 3) == 2 ? counts[2] : counts[3];
  for (int s = tid >> 2; s < total; s += THREADS / 4) {
    int at = s, from = 0;
#pragma unroll
    for (int w = 0; w < WAVES - 1; ++w) {
      const bool behind = from == w && at >= counts[w];
      at -= behind ? counts[w] : 0;
      from += behind ? 1 : 0;
    }
    const uint64_t k = left[from * WAVE_LEFT + at];
    int rank = 0;
#pragma unroll 4
    for (int t = 0; t < num_others; ++t) rank += others[t] > k;
    rank += __shfl_xor(rank, 1, VELOX_WAVE);
    rank += __shfl_xor(rank, 2, VELOX_WAVE);
    if ((tid & 3) == 0 && rank < keep) out[rank] = Candidate{from_ordered((uint32_t)(k >> 32)), base + (int)~(uint32_t)k};
  }
  for (int r = total + tid; r < keep; r += THREADS) out[r] = Candidate{-INFINITY, -1};
  if (tid == 0) {
    double all = 0.0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) all += moved_sum(wave_sums[w], wave_refs[w], top);
    sums[(size_t)row * pieces + piece] = PieceSum{all, top, 0};
  }
}

// What comes first: the greater value; of equal ones the lower beam, in one beam the greater logit (64 bits of a value need not tell two
// logits apart), then the lower token.  The second to the fourth are one number, smaller for what comes first.
struct Place { double value; uint64_t after; };
__device__ __forceinline__ uint64_t after_of(int beam, float logit, int token) {
  return (uint64_t)beam << 56 | (uint64_t)(~ordered_bits(logit)) << 24 | (uint64_t)token;
}
__device__ __forceinline__ bool before(const Place& a, const Place& b) { return a.value > b.value || (a.value == b.value && a.after < b.after); }
constexpr int MOST_BEAMS = 256, MOST_VOCAB = 1 << 24;

// Grid (requests).  All candidates' values are worked out, and the `keep` best found by counting: a bound that at least `keep` and hardly
// more candidates reach is looked for from the best value down in steps that double, then by halving the interval that is left, as a
// number whose order is the values' (64 bits), and should too many have the very same value, among those by what else decides.  What the
// bound leaves is ranked.  (Bounds from the lists' first entries alone leave nearly everything where the beams' scores lie far apart.)
// (Few candidates are four waves' work: a count is a barrier, and its time goes by the waves that meet there: 2,400 candidates 8.5 us in sixteen waves, 1,216 in four 6.4.)
constexpr int JOIN_HELD = 8;   // candidates a thread keeps in registers; the others' values lie in memory
constexpr int JOIN_LEFT = 2 * MOST_KEPT + 64;

__device__ __forceinline__ uint64_t ordered_bits_64(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
  return b ^ ((uint64_t)((long long)b >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double from_ordered_64(uint64_t o) { return __longlong_as_double((long long)((o >> 63) != 0 ? o ^ 0x8000000000000000ull : ~o)); }

template <int JOIN_THREADS>
__global__ void __launch_bounds__(JOIN_THREADS) beam_join_kernel(const float* __restrict__ scores, const PieceSum* __restrict__ sums, const Candidate* __restrict__ candidates,
                                                                 int beams, int keep, int pieces, uint64_t* __restrict__ values, float* __restrict__ out_scores,
                                                                 int* __restrict__ out_parents, int* __restrict__ out_tokens) {
  constexpr int JOIN_WAVES = JOIN_THREADS / 64;
  __shared__ Place left[JOIN_LEFT];
  __shared__ double offsets[MOST_BEAMS], tops[MOST_BEAMS];
  __shared__ float beam_scores[MOST_BEAMS];
  __shared__ __attribute__((aligned(16))) int counts[2][JOIN_WAVES];
  __shared__ uint64_t wave_best[JOIN_WAVES];
  __shared__ int num_left;
  const int request = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const size_t row0 = (size_t)request * beams;
  const int per_beam = pieces * keep, total = beams * per_beam;  // (below 2^31: the launcher sees to it)
  const Candidate* const mine = candidates + row0 * per_beam;
  uint64_t* const rest = values + row0 * per_beam;
  // (asked for before the sums: they are on nobody's way)
  Candidate held[JOIN_HELD];
#pragma unroll
  for (int k = 0; k < JOIN_HELD; ++k) {
    const int at = tid + k * JOIN_THREADS;
    held[k] = at < total ? mine[at] : Candidate{-INFINITY, -1};
  }
  // a beam's maximum, and minus the logarithm of its sum: sixteen lanes to a beam
  for (int w = tid >> 4; w < beams; w += JOIN_THREADS / 16) {
    const int first = tid & 15;
    const PieceSum* s = sums + (row0 + w) * pieces;
    const PieceSum own = first < pieces ? s[first] : PieceSum{0.0, -INFINITY, 0};
    const float score = scores[row0 + w];
    float top = own.top;
    for (int p = 16 + first; p < pieces; p += 16) top = fmaxf(top, s[p].top);
    top = over_row(top, [](float a, float b) { return fmaxf(a, b); });
    auto part = [&](const PieceSum& x) { return moved_sum(x.sum, x.top, top); };
    double sum = part(own);
    for (int p = 16 + first; p < pieces; p += 16) sum += part(s[p]);
    sum = over_row_64(sum, Sum64());
    if (first == 0) {
      tops[w] = (double)top;
      offsets[w] = top > -INFINITY ? -log(sum) : 0.0;
      beam_scores[w] = score;
    }
  }
  if (tid == 0) num_left = 0;
  __syncthreads();
  auto beam_of = [&](int at) { return (int)((unsigned)at / (unsigned)per_beam); };
  auto key_of = [&](int at, const Candidate& c) -> uint64_t {  // 0: no candidate
    if (c.token < 0) return 0;
    const int w = beam_of(at);
    const double score = (double)beam_scores[w], top = tops[w];
    const double value = score + (((double)c.logit == top ? 0.0 : (double)c.logit - top) + offsets[w]);
    return ordered_bits_64(c.logit > -INFINITY && score > -INFINITY && value >= -INFINITY ? value : -INFINITY);  // (an infinite score less infinity is none)
  };
  uint64_t key[JOIN_HELD], best = 0;
#pragma unroll
  for (int k = 0; k < JOIN_HELD; ++k) {
    key[k] = key_of(tid + k * JOIN_THREADS, held[k]);
    best = key[k] > best ? key[k] : best;
  }
  for (int at = tid + JOIN_HELD * JOIN_THREADS; at < total; at += JOIN_THREADS) {
    const uint64_t k = key_of(at, mine[at]);
    rest[at] = k;  // (read again by this thread alone)
    best = k > best ? k : best;
  }
  best = over_wave_64(best, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
  if (lane == 0) wave_best[wave] = best;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < JOIN_WAVES; ++w) best = wave_best[w] > best ? wave_best[w] : best;

  int turn = 0;
  auto count_of = [&](auto reaches) -> int {  // reaches(key, place among the candidates)
    int own = 0;
#pragma unroll
    for (int k = 0; k < JOIN_HELD; ++k) own += __popcll(__ballot(reaches(key[k], tid + k * JOIN_THREADS)));
    for (int base = JOIN_HELD * JOIN_THREADS; base < total; base += JOIN_THREADS) {
      const int at = base + tid;
      own += __popcll(__ballot(at < total && reaches(rest[at < total ? at : total - 1], at)));
    }
    turn ^= 1;
    if (lane == 0) counts[turn][wave] = own;
    __syncthreads();
    int sum = 0;
#pragma unroll
    for (int w = 0; w < JOIN_WAVES; ++w) sum += counts[turn][w];
    return sum;
  };
  // at least `keep` candidates have lo, fewer have hi; of a value of -inf and of places without a candidate: lo = 1 is what all have
  const int most = 2 * keep + 16;
  uint64_t lo = 1, hi = best + 1;
  int have = total;
  const double top_value = from_ordered_64(best);
  if (top_value > -INFINITY && top_value < INFINITY) {
    for (double below = 2.0; below <= 1024.0; below *= 2.0) {
      const uint64_t trial = ordered_bits_64(top_value - below);
      const int count = count_of([&](uint64_t k, int) { return k >= trial; });
      if (count >= keep) {
        lo = trial;
        have = count;
        break;
      }
      hi = trial;
    }
  }
  while (have > most && hi - lo > 1) {
    const uint64_t trial = lo + (hi - lo) / 2;
    const int count = count_of([&](uint64_t k, int) { return k >= trial; });
    if (count >= keep) {
      lo = trial;
      have = count;
    } else {
      hi = trial;
    }
  }
  // of those with the value lo itself only the ones up to `until` (by after_of)
  auto after_at = [&](int at) { const Candidate c = mine[at]; return after_of(beam_of(at), c.logit, c.token); };
  uint64_t until = ~0ull;
  if (have > most) {
    const int above = count_of([&](uint64_t k, int) { return k > lo; });
    uint64_t from = 0;  // fewer than are missing lie before or at it, or none
    while (have > most && until - from > 1) {
      const uint64_t trial = from + (until - from) / 2;
      const int count = above + count_of([&](uint64_t k, int at) { return k == lo && after_at(at) <= trial; });
      if (count >= keep) {
        until = trial;
        have = count;
      } else {
        from = trial;
      }
    }
  }
  auto offer = [&](uint64_t k, int at) {
    if (k < lo) return;
    const uint64_t after = after_at(at);
    if (k == lo && after > until) return;
    const int to = atomicAdd(&num_left, 1);
    if (to < JOIN_LEFT) left[to] = Place{from_ordered_64(k), after};
  };
#pragma unroll
  for (int k = 0; k < JOIN_HELD; ++k) offer(key[k], tid + k * JOIN_THREADS);
  for (int at = tid + JOIN_HELD * JOIN_THREADS; at < total; at += JOIN_THREADS) offer(rest[at], at);
  __syncthreads();
  // eight threads to a place, each with an eighth of the others
  const int count = min(num_left, JOIN_LEFT);
  for (int s = tid >> 3; s < count; s += JOIN_THREADS / 8) {
    const Place place = left[s];
    int rank = 0;
#pragma unroll 4
    for (int t = tid & 7; t < count; t += 8) rank += before(left[t], place);
    rank += __shfl_xor(rank, 1, VELOX_WAVE);
    rank += __shfl_xor(rank, 2, VELOX_WAVE);
    rank += __shfl_xor(rank, 4, VELOX_WAVE);
    if ((tid & 7) != 0 || rank >= keep) continue;
    const size_t at = (size_t)request * keep + rank;
    out_scores[at] = (float)place.value;
    out_parents[at] = (int)(place.after >> 56);
    out_tokens[at] = (int)(place.after & 0xffffffu);
  }
}

extern "C" int velox_beam_most_kept() { return MOST_KEPT; }
extern "C" int velox_beam_most_beams() { return MOST_BEAMS; }
extern "C" int velox_beam_most_vocab() { return MOST_VOCAB; }
extern "C" long long velox_beam_scratch_bytes(int rows, int pieces, int keep) {
  return (long long)rows * pieces * ((long long)sizeof(PieceSum) + (long long)keep * (sizeof(uint64_t) + sizeof(Candidate)));
}
// outputs: [requests][keep] each of values (float32), beams and tokens (int32), one behind the other
extern "C" int velox_beam_select(const float* logits, const float* scores, int requests, int beams, int vocab, int keep, int pieces, void* scratch,
                                 long long scratch_bytes, float* outputs, hipStream_t stream) {
  if (requests <= 0) return 0;
  const long long rows = (long long)requests * beams;
  if (beams < 1 || beams > MOST_BEAMS || vocab < 1 || vocab > MOST_VOCAB || keep < 1 || keep > MOST_KEPT || pieces < 1) return -1;
  if (rows > 65535 || keep > (long long)beams * vocab || (long long)beams * pieces * keep > 0x7fff0000LL) return -1;
  if (scratch_bytes < velox_beam_scratch_bytes((int)rows, pieces, keep)) return -1;
  PieceSum* const sums = (PieceSum*)scratch;
  uint64_t* const values = (uint64_t*)(sums + rows * pieces);
  Candidate* const candidates = (Candidate*)(values + rows * pieces * keep);
  const dim3 grid(pieces, (unsigned)rows);
  const int span = ((vocab + pieces - 1) / pieces + 3) / 4 * 4;  // (the last ones may be short, or have nothing)
  if (span <= 2 * 4 * THREADS) beam_pieces_kernel<2><<<grid, THREADS, 0, stream>>>(logits, scores, vocab, span, keep, pieces, sums, candidates);
  else beam_pieces_kernel<4><<<grid, THREADS, 0, stream>>>(logits, scores, vocab, span, keep, pieces, sums, candidates);
  const int status = (int)hipGetLastError();
  if (status != 0) return status;
  auto join = (long long)beams * pieces * keep <= 256 * JOIN_HELD ? beam_join_kernel<256> : beam_join_kernel<1024>;
  join<<<requests, (long long)beams * pieces * keep <= 256 * JOIN_HELD ? 256 : 1024, 0, stream>>>(scores, sums, candidates, beams, keep, pieces, values, outputs,
                                                                                              (int*)outputs + (size_t)requests * keep,
                                                                                              (int*)outputs + 2 * (size_t)requests * keep);
  return (int)hipGetLastError();
}

// ---- rows that change places -------------------------------------------------------------------------------------------------
constexpr int MOST_TENSORS = 32, MOST_MOVED = 64;
struct MovedTensor {
  char* base;
  long long outer_bytes, row_bytes;  // of one of `outer` runs of rows, of a row
  int outer_before, rows;            // outer runs of the tensors before this one
};
struct MovedTensors { MovedTensor of[MOST_TENSORS]; };

// Grid (columns, request and place, outer runs of all tensors); a column is as many bytes as a Column.  Every row that anybody takes over is
// read once, whoever takes it.  Bound by memory: 8 requests of 8 beams, 16 runs of rows of 512 KiB, 813 MB read and written in 147 to 152 us, 5.4 TB/s (a copy
// reaches 4.8); reading a row anew for every beam that takes it was 280.
template <typename Column, int MOST>
__global__ void __launch_bounds__(THREADS, MOST <= 8 ? 8 : MOST <= 16 ? 4 : MOST <= 32 ? 2 : 1)
reorder_kernel(const MovedTensors tensors, int count, const int* __restrict__ slots, const int* __restrict__ parents, int beams, int places) {
  int at = 0;
  for (int t = 1; t < count; ++t) at = (int)blockIdx.z >= tensors.of[t].outer_before ? t : at;
  const MovedTensor tensor = tensors.of[at];
  if ((long long)blockIdx.x * THREADS * (long long)sizeof(Column) >= tensor.row_bytes) return;
  const long long column = ((long long)blockIdx.x * THREADS + threadIdx.x) * (long long)sizeof(Column);
  const int request = blockIdx.y / places, place = blockIdx.y % places, lane = threadIdx.x & 63;
  // lane j: beam j's parent, its row, and whether it takes over another one
  int parent = -1, row = -1;
  if (lane < beams) {
    parent = parents[(long long)request * beams + lane];
    row = slots[((long long)request * beams + lane) * places + place];
  }
  const bool there = row >= 0 && row < tensor.rows;
  const uint64_t rows_there = __ballot(there);
  const int source = __shfl(row, parent & 63, VELOX_WAVE);  // (by all lanes: what a lane that stood out had would not be read)
  const bool moves = there && parent >= 0 && parent < beams && (rows_there >> (parent & 63) & 1) != 0 && source != row;
  uint64_t taken = 0;
  for (uint64_t left = __ballot(moves); left != 0; left &= left - 1) taken |= 1ull << __builtin_amdgcn_readlane(parent, __ffsll((unsigned long long)left) - 1);
  if (taken == 0) return;
  const bool live = column < tensor.row_bytes;
  char* const base = tensor.base + (long long)((int)blockIdx.z - tensor.outer_before) * tensor.outer_bytes + column;
  auto row_at = [&](int beam) { return base + (long long)__builtin_amdgcn_readlane(row, beam) * tensor.row_bytes; };
  Column held[MOST];
  uint64_t todo = taken;
#pragma unroll
  for (int k = 0; k < MOST; ++k) {
    if (todo != 0) {
      if (live) held[k] = __builtin_nontemporal_load(reinterpret_cast<const Column*>(row_at(__ffsll((unsigned long long)todo) - 1)));
      todo &= todo - 1;
    }
  }
  todo = taken;
#pragma unroll
  for (int k = 0; k < MOST; ++k) {
    if (todo != 0) {
      for (uint64_t to = __ballot(moves && parent == __ffsll((unsigned long long)todo) - 1); to != 0; to &= to - 1)
        if (live) __builtin_nontemporal_store(held[k], reinterpret_cast<Column*>(row_at(__ffsll((unsigned long long)to) - 1)));
      todo &= todo - 1;
    }
  }
}

extern "C" int velox_reorder_most_tensors() { return MOST_TENSORS; }
extern "C" int velox_reorder_most_beams() { return MOST_MOVED; }

template <typename Column>
static int launch_reorder(const MovedTensors& tensors, int count, long long widest, int outer, const int* slots, const int* parents, int requests, int beams, int places,
                          hipStream_t stream) {
  const long long blocks = (widest + THREADS * (long long)sizeof(Column) - 1) / (THREADS * (long long)sizeof(Column));
  if (blocks > 0x7fffffffLL) return -1;
  const dim3 grid((unsigned)blocks, (unsigned)(requests * places), (unsigned)outer);
  if (beams <= 4) reorder_kernel<Column, 4><<<grid, THREADS, 0, stream>>>(tensors, count, slots, parents, beams, places);
  else if (beams <= 8) reorder_kernel<Column, 8><<<grid, THREADS, 0, stream>>>(tensors, count, slots, parents, beams, places);
  else if (beams <= 16) reorder_kernel<Column, 16><<<grid, THREADS, 0, stream>>>(tensors, count, slots, parents, beams, places);
  else if (beams <= 32) reorder_kernel<Column, 32><<<grid, THREADS, 0, stream>>>(tensors, count, slots, parents, beams, places);
  else reorder_kernel<Column, 64><<<grid, THREADS, 0, stream>>>(tensors, count, slots, parents, beams, places);
  return (int)hipGetLastError();
}

// described: per tensor its address, its outer runs, the bytes of a run, its rows, the bytes of a row (five numbers each, on the host).
extern "C" int velox_reorder_states(const long long* described, int count, const int* slots, const int* parents, int requests, int beams, int places, hipStream_t stream) {
  if (requests <= 0 || places <= 0 || count <= 0) return 0;
  if (count > MOST_TENSORS || beams < 1 || beams > MOST_MOVED || (long long)requests * places > 65535) return -1;
  MovedTensors tensors = {};
  long long outer = 0, widest = 0, bits = 0;
  for (int t = 0; t < count; ++t) {
    const long long* d = described + 5 * t;
    if (d[1] < 0 || d[3] < 0 || d[3] > 0x7fffffffLL || d[4] < 0) return -1;
    tensors.of[t] = MovedTensor{(char*)(uintptr_t)d[0], d[2], d[4], (int)outer, (int)d[3]};
    outer += d[1];
    if (outer > 65535) return -1;
    widest = d[4] > widest ? d[4] : widest;
    bits |= d[0] | d[2] | d[4];
  }
  if (outer == 0 || widest == 0) return 0;
  if (bits % 16 == 0) return launch_reorder<float4_t>(tensors, count, widest, (int)outer, slots, parents, requests, beams, places, stream);
  if (bits % 4 == 0) return launch_reorder<uint32_t>(tensors, count, widest, (int)outer, slots, parents, requests, beams, places, stream);
  if (bits % 2 == 0) return launch_reorder<uint16_t>(tensors, count, widest, (int)outer, slots, parents, requests, beams, places, stream);
  return launch_reorder<uint8_t>(tensors, count, widest, (int)outer, slots, parents, requests, beams, places, stream);
}
