// Several continuations of one request (beams) for gfx950: which of them go on, and what they held moving with them.
//
// beam_select.  Beam w of a request stands at scores[w]; a continuation by token v is worth
//     value(w, v) = scores[w] + (logits[w, v] - max_w - log sum_u exp(logits[w, u] - max_w)),
// and the `keep` most valuable of all beams and tokens are wanted, best first, ties to the lowest (w, v).  Within a beam the order is the
// logits' own, so a row's best `keep` hold all that can be wanted of it; what decides between rows is the log-sum, in which a rounding to 32
// bits would change the order of near ones: sums and values are held in 64 bits.  One kernel reads the logits once, a piece of a row per
// workgroup, and leaves each piece's maximum, sum of exponentials and best `keep` in order; a second, one workgroup per request, joins them.
//
// A piece's best `keep`.  Every value gets a key that no other of the piece has: its bits in an order that compares like numbers, then
// its place counted from the end.  The `keep`-th largest among the maxima of disjoint parts of the piece is not above the `keep`-th
// largest key of all, and at most `keep` parts hold keys as large: only those keys, a few more than `keep` as a rule, are ranked.
//
// reorder_states: row slots[b, j, p] of every tensor becomes what row slots[b, parents[b, j], p] was.  A thread owns a column of the rows of one
// request: it has read all that move before it writes any, and nobody else reads or writes that column, so the rows change places
// in the memory they are in.
#include "common.h"

// ---- selection ------------------------------------------------------------------------------------------------------------
constexpr int THREADS = 256;
constexpr int MOST_KEPT = 64;

// exp(x) for x <= 0 in 64 bits, to 1e-11 of it: x = k ln 2 + r with |r| <= ln 2 / 2, and the series of e^r to its ninth power
// (the next term is at most 0.347^10 / 10! = 7e-12).
__device__ __forceinline__ double exp_below_zero(double x) {
  const double k = rint(x * 1.4426950408889634074);
  const double r = fma(k, -0.69314718055994530942, x);
  double e = 1.0 / 362880.0;
  e = fma(e, r, 1.0 / 40320.0);
  e = fma(e, r, 1.0 / 5040.0);
  e = fma(e, r, 1.0 / 720.0);
  e = fma(e, r, 1.0 / 120.0);
  e = fma(e, r, 1.0 / 24.0);
  e = fma(e, r, 1.0 / 6.0);
  e = fma(e, r, 0.5);
  e = fma(e, r, 1.0);
  e = fma(e, r, 1.0);
  return x < -700.0 ? 0.0 : ldexp(e, (int)k);
}

__device__ __forceinline__ uint32_t ordered_bits(float v) {  // compares like the number
  const uint32_t b = __float_as_uint(v);
  return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t o) { return __uint_as_float((o & 0x80000000u) != 0 ? o ^ 0x80000000u : ~o); }

__device__ __forceinline__ double wave_sum_64(double v) {
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1) v += __shfl_xor(v, offset, VELOX_WAVE);
  return v;
}

struct PieceSum { double sum; float top; int unused; };  // sum of exp(logit - top)
struct Candidate { float logit; int token; };            // token < 0: none

// Grid (pieces, rows).  sums: [row][piece]; candidates: [row][piece][keep], best first.
template <int PER_THREAD>
__global__ void __launch_bounds__(THREADS) beam_pieces_kernel(const float* __restrict__ logits, const float* __restrict__ scores, int vocab, int keep, int pieces,
                                                              PieceSum* __restrict__ sums, Candidate* __restrict__ candidates) {
  constexpr int PIECE = THREADS * PER_THREAD, QUADS = PER_THREAD / 4;
  constexpr int PLACE_BITS = 13;
  static_assert(PIECE <= 1 << PLACE_BITS, "a place of the piece fits its bits");
  constexpr int MOST_LEFT = 32 * 4 * PER_THREAD;  // keys that may be left to rank: 32 parts of four threads, or 64 of one
  __shared__ uint64_t left[MOST_LEFT];
  __shared__ uint64_t part_best[THREADS];
  __shared__ float wave_tops[THREADS / 64];
  __shared__ double wave_sums[THREADS / 64];
  __shared__ int num_left;

  const int row = blockIdx.y, piece = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  Candidate* const out = candidates + ((size_t)row * pieces + piece) * keep;
  if (!(scores[row] > -INFINITY)) {  // a beam that is not there: its continuations are all alike, the first tokens come first
    for (int r = tid; r < keep; r += THREADS) out[r] = Candidate{-INFINITY, piece == 0 && r < vocab ? r : -1};
    if (tid == 0) sums[(size_t)row * pieces + piece] = PieceSum{0.0, -INFINITY, 0};
    return;
  }
  // (a row begins wherever the one before ends: loads of four numbers at any multiple of four bytes.  Which thread adds up which tokens
  // must not hang on that, or equal rows would differ in their sums' last bits)
  typedef float loose4_t __attribute__((ext_vector_type(4), aligned(4)));
  const float* const first = logits + (size_t)row * vocab;
  const int base = piece * PIECE;  // the piece's first token
  float v[PER_THREAD];
#pragma unroll
  for (int q = 0; q < QUADS; ++q) {
    const int token = base + 4 * (q * THREADS + tid);
    if (token + 4 <= vocab) {
      const loose4_t x = *reinterpret_cast<const loose4_t*>(first + token);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * q + j] = x[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * q + j] = token + j < vocab ? first[token + j] : -INFINITY;
    }
  }
  if (tid == 0) num_left = 0;
  float top = -INFINITY;
#pragma unroll
  for (int e = 0; e < PER_THREAD; ++e) {
    v[e] = v[e] == v[e] ? v[e] + 0.f : -INFINITY;  // (no number: never chosen before one; a zero has one form)
    top = fmaxf(top, v[e]);
  }
  // keys: value, then place from the end; 0 for places outside the row
  auto key_of = [&](int e) -> uint64_t {
    const int place = 4 * ((e >> 2) * THREADS + tid) + (e & 3), token = base + place;
    return token < vocab ? ((uint64_t)ordered_bits(v[e]) << PLACE_BITS) | (uint64_t)((1 << PLACE_BITS) - 1 - place) : 0;
  };
  uint64_t best = 0;
#pragma unroll
  for (int e = 0; e < PER_THREAD; ++e) {
    const uint64_t k = key_of(e);
    best = k > best ? k : best;
  }
  part_best[tid] = best;
  const float wave_top = wave_max(top);
  if (lane == 0) wave_tops[wave] = wave_top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) top = fmaxf(top, wave_tops[w]);
  double sum = 0.0;
  if (top > -INFINITY) {
    const double ref = (double)top;
#pragma unroll
    for (int e = 0; e < PER_THREAD; ++e) sum += v[e] == top ? 1.0 : exp_below_zero(top < INFINITY ? (double)v[e] - ref : -INFINITY);
  }
  sum = wave_sum_64(sum);
  if (lane == 0) wave_sums[wave] = sum;
  // The bound: parts are single threads, or four of them while 64 parts are twice `keep`.  A wave finds the `keep`-th largest of the
  // maxima bit by bit from the highest down; with fewer parts than `keep` that hold anything it is what all keys exceed.
  uint64_t bound = 0;
  {
    uint64_t k[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) k[a] = part_best[64 * a + lane];
    if (keep <= 32) {
#pragma unroll
      for (int a = 1; a < 4; ++a) {
        k[0] = k[a] > k[0] ? k[a] : k[0];
        k[a] = 0;
      }
    }
    for (int bit = 32 + PLACE_BITS - 1; bit >= 0; --bit) {
      const uint64_t trial = bound | 1ull << bit;
      int count = 0;
#pragma unroll
      for (int a = 0; a < 4; ++a) count += __popcll(__ballot(k[a] >= trial));
      if (count >= keep) bound = trial;
    }
  }
  bound = bound > 0 ? bound : 1;
  __syncthreads();  // (num_left is set)
#pragma unroll
  for (int e = 0; e < PER_THREAD; ++e) {
    const uint64_t k = key_of(e);
    if (k >= bound) {
      const int at = atomicAdd(&num_left, 1);
      if (at < MOST_LEFT) left[at] = k;
    }
  }
  __syncthreads();
  const int count = min(num_left, MOST_LEFT);
  for (int s = tid; s < count; s += THREADS) {
    const uint64_t k = left[s];
    int rank = 0;
    for (int t = 0; t < count && rank < keep; ++t) rank += left[t] > k;
    if (rank < keep) out[rank] = Candidate{from_ordered((uint32_t)(k >> PLACE_BITS)), base + (1 << PLACE_BITS) - 1 - (int)(k & ((1 << PLACE_BITS) - 1))};
  }
  for (int r = count + tid; r < keep; r += THREADS) out[r] = Candidate{-INFINITY, -1};
  if (tid == 0) {
    double total = 0.0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) total += wave_sums[w];
    sums[(size_t)row * pieces + piece] = PieceSum{total, top, 0};
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

// Grid (requests).  A list is a piece's candidates in order, `beams * pieces` of them.  Of the lists' first ones the `keep`-th best is a
// bound: no list whose first lies behind it holds anything that is wanted, and at most `keep` lists do not.
constexpr int JOIN_THREADS = 1024;
constexpr int JOIN_LEFT = MOST_KEPT * MOST_KEPT;
__global__ void __launch_bounds__(JOIN_THREADS) beam_join_kernel(const float* __restrict__ scores, const PieceSum* __restrict__ sums, const Candidate* __restrict__ candidates,
                                                                 int beams, int keep, int pieces, float* __restrict__ out_scores, int* __restrict__ out_parents,
                                                                 int* __restrict__ out_tokens) {
  __shared__ Place left[JOIN_LEFT];  // (the lists' firsts before)
  __shared__ double offsets[MOST_BEAMS], tops[MOST_BEAMS];
  __shared__ Place limit;
  __shared__ int num_left;
  const int request = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const size_t row0 = (size_t)request * beams;
  const int lists = beams * pieces;
  const Place last = {-INFINITY, ~0ull};
  // a beam's maximum, and minus the logarithm of its sum
  for (int w = wave; w < beams; w += JOIN_THREADS / 64) {
    const PieceSum* s = sums + (row0 + w) * pieces;
    float top = -INFINITY;
    for (int p = lane; p < pieces; p += 64) top = fmaxf(top, s[p].top);
    top = wave_max(top);
    double sum = 0.0;
    for (int p = lane; p < pieces; p += 64) {
      const PieceSum x = s[p];
      if (x.top > -INFINITY) sum += x.top == top ? x.sum : x.sum * exp_below_zero(top < INFINITY ? (double)x.top - (double)top : -INFINITY);
    }
    sum = wave_sum_64(sum);
    if (lane == 0) {
      tops[w] = (double)top;
      offsets[w] = top > -INFINITY ? -log(sum) : 0.0;
    }
  }
  if (tid == 0) {
    num_left = 0;
    limit = last;
  }
  __syncthreads();
  const Candidate* const mine = candidates + row0 * pieces * keep;
  auto place_of = [&](int w, const Candidate& c) -> Place {
    const float score = scores[row0 + w];
    const double top = tops[w];
    const double value = !(c.logit > -INFINITY) || !(score > -INFINITY) ? -INFINITY : (double)score + (((double)c.logit == top ? 0.0 : (double)c.logit - top) + offsets[w]);
    return Place{value, after_of(w, c.logit, c.token)};
  };
  auto first_of = [&](int a) -> Place {
    if (a >= lists) return last;
    const Candidate c = mine[(size_t)a * keep];
    return c.token >= 0 ? place_of(a / pieces, c) : last;
  };
  if (lists >= keep) {
    for (int a0 = 0; a0 < lists; a0 += JOIN_THREADS) {
      const Place own = first_of(a0 + tid);
      int rank = 0;
      for (int o0 = 0; o0 < lists; o0 += JOIN_THREADS) {
        __syncthreads();
        left[tid] = o0 == a0 ? own : first_of(o0 + tid);
        __syncthreads();
        const int here = min(lists - o0, JOIN_THREADS);
        for (int o = 0; o < here; ++o) rank += before(left[o], own);
      }
      if (rank == keep - 1 && own.after != last.after) limit = own;
    }
  }
  __syncthreads();
  const Place bound = limit;
  for (int a = tid; a < lists; a += JOIN_THREADS) {
    const int w = a / pieces;
    for (int r = 0; r < keep; ++r) {
      const Candidate c = mine[(size_t)a * keep + r];
      if (c.token < 0) break;
      const Place place = place_of(w, c);
      if (before(bound, place)) break;  // (the list is in order)
      const int at = atomicAdd(&num_left, 1);
      if (at < JOIN_LEFT) left[at] = place;
    }
  }
  __syncthreads();
  const int count = min(num_left, JOIN_LEFT);
  for (int s = tid; s < count; s += JOIN_THREADS) {
    const Place place = left[s];
    int rank = 0;
    for (int t = 0; t < count && rank < keep; ++t) rank += before(left[t], place);
    if (rank >= keep) continue;
    const size_t at = (size_t)request * keep + rank;
    out_scores[at] = (float)place.value;
    out_parents[at] = (int)(place.after >> 56);
    out_tokens[at] = (int)(place.after & 0xffffffu);
  }
}

extern "C" int velox_beam_most_kept() { return MOST_KEPT; }
extern "C" int velox_beam_most_beams() { return MOST_BEAMS; }
extern "C" int velox_beam_most_vocab() { return MOST_VOCAB; }
// pieces of a row; `per_thread` is 8 or 32
extern "C" int velox_beam_pieces(int vocab, int per_thread) { return (vocab + THREADS * per_thread - 1) / (THREADS * per_thread); }
extern "C" long long velox_beam_scratch_bytes(int rows, int pieces, int keep) {
  return (long long)rows * pieces * ((long long)sizeof(PieceSum) + (long long)keep * sizeof(Candidate));
}
extern "C" int velox_beam_select(const float* logits, const float* scores, int requests, int beams, int vocab, int keep, int per_thread, void* scratch,
                                 long long scratch_bytes, float* out_scores, int* out_parents, int* out_tokens, hipStream_t stream) {
  if (requests <= 0) return 0;
  const int pieces = velox_beam_pieces(vocab, per_thread);
  const long long rows = (long long)requests * beams;
  if (beams < 1 || beams > MOST_BEAMS || vocab < 1 || vocab > MOST_VOCAB || keep < 1 || keep > MOST_KEPT || (per_thread != 8 && per_thread != 32)) return -1;
  if (rows > 65535 || keep > (long long)beams * vocab) return -1;
  if (scratch_bytes < velox_beam_scratch_bytes((int)rows, pieces, keep)) return -1;
  PieceSum* const sums = (PieceSum*)scratch;
  Candidate* const candidates = (Candidate*)(sums + rows * pieces);
  const dim3 grid(pieces, (unsigned)rows);
  if (per_thread == 8) beam_pieces_kernel<8><<<grid, THREADS, 0, stream>>>(logits, scores, vocab, keep, pieces, sums, candidates);
  else beam_pieces_kernel<32><<<grid, THREADS, 0, stream>>>(logits, scores, vocab, keep, pieces, sums, candidates);
  const int status = (int)hipGetLastError();
  if (status != 0) return status;
  beam_join_kernel<<<requests, JOIN_THREADS, 0, stream>>>(scores, sums, candidates, beams, keep, pieces, out_scores, out_parents, out_tokens);
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

// Grid (columns, request and place, outer runs of all tensors); a column is WIDTH bytes.
template <typename Column, int MOST>
__global__ void __launch_bounds__(THREADS) reorder_kernel(const MovedTensors tensors, int count, const int* __restrict__ slots, const int* __restrict__ parents, int beams,
                                                          int places) {
  int at = 0;
  for (int t = 1; t < count; ++t) at = (int)blockIdx.z >= tensors.of[t].outer_before ? t : at;
  const MovedTensor tensor = tensors.of[at];
  const long long column = ((long long)blockIdx.x * THREADS + threadIdx.x) * (long long)sizeof(Column);
  if ((long long)blockIdx.x * THREADS * (long long)sizeof(Column) >= tensor.row_bytes) return;
  const int request = blockIdx.y / places, place = blockIdx.y % places, lane = threadIdx.x & 63;
  // lane j: where beam j's row lies and where its parent's does
  int row = -1, from = -1;
  if (lane < beams) {
    row = slots[((long long)request * beams + lane) * places + place];
    const int parent = parents[(long long)request * beams + lane];
    from = parent >= 0 && parent < beams ? slots[((long long)request * beams + parent) * places + place] : -1;
  }
  uint64_t moving = __ballot(row >= 0 && row < tensor.rows && from >= 0 && from < tensor.rows && from != row);
  if (column >= tensor.row_bytes) return;
  char* const base = tensor.base + (long long)((int)blockIdx.z - tensor.outer_before) * tensor.outer_bytes + column;
  Column held[MOST];
  uint64_t todo = moving;
#pragma unroll
  for (int k = 0; k < MOST; ++k) {
    if (todo != 0) {
      const int j = __ffsll((unsigned long long)todo) - 1;
      todo &= todo - 1;
      held[k] = *reinterpret_cast<const Column*>(base + (long long)__builtin_amdgcn_readlane(from, j) * tensor.row_bytes);
    }
  }
  todo = moving;
#pragma unroll
  for (int k = 0; k < MOST; ++k) {
    if (todo != 0) {
      const int j = __ffsll((unsigned long long)todo) - 1;
      todo &= todo - 1;
      *reinterpret_cast<Column*>(base + (long long)__builtin_amdgcn_readlane(row, j) * tensor.row_bytes) = held[k];
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
