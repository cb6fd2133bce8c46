// Attention of single tokens over a paged cache for gfx950, for sequences that share their first keys in groups; one head size
// per build (-DVELOX_HEAD_DIM=<multiple of 16>), float32 and bfloat16.
//
// Sequence b brings one token that sees its kv_lens[b] keys.  Group g is the sequences group_starts[g] .. group_starts[g + 1] - 1,
// whose first shared_lens[g] keys are the same ones in the same pages.  With the query heads of a KV head G:
//
//   o = sum_n exp(s_n - m) v_n / sum_n exp(s_n - m),   s_n = scale q . k_n,   split as  n < P  and  n >= P
//
// for any split point P: each part gives its own o and log-sum l, and o = sum_i exp(l_i) o_i / sum_i exp(l_i).  The first part's keys
// are the same for the group's sequences, so n_g G rows of queries stand against one stream of keys and values, which is read
// once for every block of 16 (float32, and heads of more than 128 channels), 32 or 128 of them; the second part is each sequence's own, G rows
// against its keys.
//
// Four kernels; which ones a call takes goes by its sizes (the host's rules):
//
//   few keys        a workgroup per (KV head, sequence, 16 rows) takes all of its keys, nothing is shared out (shared_prefix_direct_kernel)
//   else            both parts are cut into items of about equally many keys, all in one launch, and a second kernel joins what the items leave;
//                   with more than 64 sequences or groups a third one has worked the items out before
//
// A group's item is a workgroup's: its four waves take a tile of keys in turn, each straight from the cache into the operands of matrix
// instructions, and put their results together at the end.  A sequence's own keys are single waves' items, four of them to a workgroup.  No
// wave shares a key with another, so nothing is staged and no barrier stands in the loop: the next tile's keys are asked for as soon as
// this one's have been multiplied, its values as soon as this one's have, two workgroups to a compute unit.  With many rows the products
// count, and the waves share tiles in LDS instead (tall_item).
//
// What bounds them, measured on MI355X (bfloat16; medians of 30 traced calls, kernel by kernel: an untraced call takes up to a tenth less than their sum): 48 groups of 5
// behind 700 keys (32 heads over 8 of 64 channels, 76 MB) 5.2 + 18.8 + 4.9 us, the stream at 4.0 TB/s in the main one, 2.6 of all three; 8 groups of up to 4 behind 2,048 (28
// over 4 of 128, 31 MB) 12.0 + 4.3, four loads that wait for one another and two launches; 64 sequences behind 8,192 (28 over 4, 7.6 GFLOP) 24.6 + 6.5, of which writing and
// reading the parts' 2 x 24 MB is 8 and half a tile of rows is padding; behind 32,768 (40 over 8, 43 GFLOP) 86.6 + 8.3 (81 a call untraced, 0.53 PFLOP/s): products and weights
// alone 62, loads alone 46, the sequences' own keys, a third of the bytes, 10, of untraced copies.  4 sequences of 321 keys, taken whole, 8.3 us, in parts it was 7.4 + 3.2 and
// a launch more.
//
// Matrix cores: S^T[key, row] = K Q^T and O^T[channel, row] = V^T P^T, both with 16 x 16 results.  For a block of KB contraction
// indices (32 in bfloat16, 16 in float32) lane (g = lane / 16, i = lane % 16) holds 16 bytes of row or column i, those of place g; a result is rows
// 4 g .. 4 g + 3 of column i.  In bfloat16 row 4 q + j of the tile's score tile u (q, j < 4) is key 8 q + 4 u + j, so that a lane's
// scores of both are those of keys 8 g .. 8 g + 7: the operand of the second product, and one load of V^T.
#include <type_traits>

#include "common.h"

#ifndef VELOX_HEAD_DIM
#error "build with -DVELOX_HEAD_DIM=<head size>"
#endif
constexpr int D = VELOX_HEAD_DIM;
static_assert(D % 16 == 0 && D >= 16 && D <= 256, "head size must be a multiple of 16 between 16 and 256");

constexpr int WAVES = 4, THREADS = 64 * WAVES;
constexpr int LANE_CHANNELS = D <= 64 ? 1 : D <= 128 ? 2 : 4;                              // of the joining kernel,
constexpr int JOINED_AT_ONCE = 64 / LANE_CHANNELS < 32 ? 64 / LANE_CHANNELS : 32;          // and parts
constexpr int MOST_GROUPS = 1024, MOST_KEYS = 1 << 25;  // of a call, of a sequence

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

template <typename T> struct Block;
template <> struct Block<bf16_t> {
  static constexpr int KB = 32, VEC = 8;  // a tile of keys is one block of the second product: KB keys, KB / 16 score tiles
  static constexpr float SCALE = 1.44269504088896340736f, LN_UNIT = 0.69314718055994530942f;  // scores in powers of two
  static __device__ __forceinline__ float4_t mma(const float4_t& a, const float4_t& b, const float4_t& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x); }
  static __device__ __forceinline__ int key_row(int u, int i) { return 8 * (i >> 2) + 4 * u + (i & 3); }  // key of row i of score tile u
  static __device__ __forceinline__ int first_score(int u, int g) { return 8 * g + 4 * u; }               // key of a lane's first score of it
  static __device__ __forceinline__ void mask(float4_t& v, int from, int to) {                            // zero outside [from, to)
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t keep = (2 * w >= from && 2 * w < to ? 0x0000ffffu : 0u) | (2 * w + 1 >= from && 2 * w + 1 < to ? 0xffff0000u : 0u);
      v[w] = __uint_as_float(__float_as_uint(v[w]) & keep);
    }
  }
};
template <> struct Block<float> {
  static constexpr int KB = 16, VEC = 4;
  static constexpr float SCALE = 1.f, LN_UNIT = 1.f;
  static __device__ __forceinline__ float4_t mma(const float4_t& a, const float4_t& b, float4_t c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ float exp_of(float x) { return expf(x); }
  static __device__ __forceinline__ int key_row(int u, int i) { return 16 * u + i; }
  static __device__ __forceinline__ int first_score(int u, int g) { return 16 * u + 4 * g; }
  static __device__ __forceinline__ void mask(float4_t& v, int from, int to) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = j >= from && j < to ? v[j] : 0.f;
  }
};

// ---- which workgroup does what -----------------------------------------------------------------------------------------
// Everything is worked out from the lengths on the device, so that a captured step replays with other lengths.  A group's shared
// keys are those of its first sequence at most (it is through that one's table that they are read); a sequence with fewer keys
// than its group shares, one that is alone in its group or in none, and what a group has beyond `largest` share nothing.  A step is a tile of
// keys for each of four waves (with many rows: one of the tiles that they share); all items' steps over `target` workgroups are what one item
// may have (`per`: of a sequence's own keys, tiles of one wave).  A group's rows are cut into blocks of `block_rows`, a sequence's G rows into
// blocks of 16.
//
// What the items leave has rows of its own, per KV head: `block_rows` for every item of a group, in the order groups, parts of the keys, row blocks, then
// 16 for every item of a sequence, in the order sequences, parts, blocks.  Row r of a group's or of a sequence's part p then lies at
// start + p stride + r.
struct Directory { int shared_at, shared_stride, shared_parts, own_at, own_parts, unused[3]; };  // of a sequence: where its rows lie
struct Item {           // group >= 0: of that group's shared keys, by the whole workgroup; else sequence >= 0: of its own keys, by one wave; else none
  int group, sequence;
  int first, count;     // the group's first sequence, and how many it has
  int block, from, to;  // row block, keys
  int at;               // its rows' place
};
struct Lengths {
  const int* kv_lens;
  const int* group_starts;
  const int* shared_lens;
  const Item* planned;                                  // every wave's item, if there are more groups or sequences than a wave has lanes; or nullptr
  int num_seqs, num_groups, group, block_rows, target;  // group: query heads of a KV head
  int most;                                             // keys a table has room for
  int largest;                                          // sequences of a group
  int rows_room;
};
struct Own { int group, from, to; };  // a sequence's own keys [from, to); group: whose shared keys it has, or -1

__device__ __forceinline__ int clamped(int v, int lo, int hi) { return v < lo ? lo : (v > hi ? hi : v); }
// a / b rounded down, 0 <= a < 2^23, 1 <= b < 2^23, a / b < 2^22: by the reciprocal.  a and b are exact in 32 bits, the reciprocal is off by 2^-23 of it at most and the
// product by 2^-24 of it, the estimate so by less than 0.75, after rounding down by one at most; q b lies within b of a.
// Divided are a sequence's steps or tiles of keys and what an item has of them, together, by the latter (2^21 of either at most, an item's half more where parts
// are fitted to the units), and an item's place among those of its group or sequence, which a launch's 65,535 workgroups of four waves hold.
static_assert(MOST_KEYS / 16 * 5 / 2 < 1 << 23 && MOST_KEYS / 16 < 1 << 22 && WAVES * 65535 < 1 << 22, "numbers that the quotient takes");
__device__ __forceinline__ int quotient(int a, int b) {
  int q = (int)((float)a * __builtin_amdgcn_rcpf((float)b));
  const int rest = a - q * b;
  q += rest >= b ? 1 : 0;
  q -= rest < 0 ? 1 : 0;
  return q;
}
__device__ __forceinline__ int parts_of(int steps, int per) { return quotient(steps + per - 1, per); }

// the operation over v and those of the lanes before
#define VELOX_UP_TO_LANE(OP)                                                                           \
  OP(0x111, 0xf); /* from 1, 2, 4 and 8 lanes down in a row of 16, */                                  \
  OP(0x112, 0xf);                                                                                      \
  OP(0x114, 0xf);                                                                                      \
  OP(0x118, 0xf);                                                                                      \
  OP(0x142, 0xa); /* from the end of the row before, into the second and the fourth, */                \
  OP(0x143, 0xc); /* from the middle, into the upper half */
__device__ __forceinline__ int sum_up_to_lane(int v) {
#define VELOX_ADD_SHIFTED(CONTROL, ROWS) v += __builtin_amdgcn_update_dpp(0, v, CONTROL, ROWS, 0xf, false)
  VELOX_UP_TO_LANE(VELOX_ADD_SHIFTED)
#undef VELOX_ADD_SHIFTED
  return v;
}
__device__ __forceinline__ int most_up_to_lane(int v) {  // v >= 0
#define VELOX_MAX_SHIFTED(CONTROL, ROWS) v = max(v, __builtin_amdgcn_update_dpp(0, v, CONTROL, ROWS, 0xf, false))
  VELOX_UP_TO_LANE(VELOX_MAX_SHIFTED)
#undef VELOX_MAX_SHIFTED
  return v;
}
#undef VELOX_UP_TO_LANE

// Numbers of a plan, by the keys of a tile and of a group's step (powers of two).
struct Counts {
  int tile_shift, step_shift, block_shift, own_blocks;
  __device__ __forceinline__ Counts(const Lengths& l, int tile_shift, int step_shift)
      : tile_shift(tile_shift), step_shift(step_shift), block_shift(31 - __builtin_clz(l.block_rows)), own_blocks((l.group + 15) / 16) {}
  __device__ __forceinline__ int steps(int keys) const { return (keys + (1 << step_shift) - 1) >> step_shift; }
  __device__ __forceinline__ int tiles(const Own& own) const { return own.to > own.from ? ((own.to + (1 << tile_shift) - 1) >> tile_shift) - (own.from >> tile_shift) : 0; }
  __device__ __forceinline__ int blocks(const Lengths& l, int count, int shared) const { return shared > 0 ? (count * l.group + l.block_rows - 1) >> block_shift : 0; }
  __device__ __forceinline__ int per(const Lengths& l, int steps, int tiles) const {
    return clamped((steps + (tiles + WAVES - 1) / WAVES + l.target - 1) / l.target, 1, MOST_KEYS / 16);  // (nobody has more)
  }
  // `target` workgroups are as many as the compute units take in one go, and the first one more takes as long again; rounding parts up can bring it about.
  // Then somewhat longer parts are tried (of 6 groups of up to 13 behind 10,350 keys, 16 heads over 4, were 72 items for 64 units).
  static __device__ __forceinline__ bool fills_units(const Lengths& l) { return l.block_rows > 16 * WAVES; }
  __device__ __forceinline__ int most_parts(const Own& own) const { return tiles(own) + (own.group >= 0 ? steps(own.from) : 0); }
  // Two steps instead of one make short items twice as long: up to two workgroups a unit then have one each, if that leaves no sequence more parts than the
  // joining kernel asks for at once (5 groups of up to 8 behind 1,500 float32 keys, 12 heads over 2: 16.7 / 18.2 us; one of 10 behind 2,984 22.0 / 15.2).
  // counted(per): the groups' items, or with 0 their blocks; most_parts(): a sequence's with a step each
  template <typename Counted, typename MostParts> __device__ __forceinline__ int fitted(const Lengths& l, int per, Counted counted, MostParts most_parts) const {
    if (per == 2 && !fills_units(l) && most_parts() <= JOINED_AT_ONCE) return 1;
    if ((per < 4 && !fills_units(l)) || counted(per) <= l.target || counted(0) > l.target) return per;
    int longer = per;
    for (int tries = 0; tries < 6; ++tries) {
      longer += 1 + (longer >> 4);
      if (counted(longer) <= l.target) return longer;
    }
    return per;
  }
  __device__ __forceinline__ Item of_group(const Lengths& l, int item, int place, int group, int first, int count, int shared, int per) const {
    const int row_blocks = blocks(l, count, shared), part = quotient(place, row_blocks), from = (part * per) << step_shift;
    return Item{group, -1, first, count, place - part * row_blocks, from, min(from + (per << step_shift), shared), item << block_shift};
  }
  __device__ __forceinline__ Item of_sequence(int item, int place, int sequence, int from, int to, int per, int group_items) const {
    const int part = quotient(place, own_blocks), low = ((from >> tile_shift) + part * per) << tile_shift;
    return Item{-1, sequence, 0, 0, place - part * own_blocks, max(low, from), min(low + (per << tile_shift), to), (group_items << block_shift) + item * 16};
  }
};
__device__ __forceinline__ Own own_keys(int group, int shared, int len) { return shared > 0 && shared <= len ? Own{group, shared, len} : Own{-1, 0, len}; }

// With up to 64 sequences and groups every wave works its item out for itself: a lane has a group and a sequence of its own.  (1.7 us; with 240
// sequences, 64 at a time, it was 7 of 24.5 us, with 1,000 68 of 145.)  `begins`: this wave's 64 places in LDS.
__device__ __forceinline__ Item find_item(const Lengths& l, const Counts& counts, int wg, int* begins, Directory* __restrict__ directory) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  auto at_most = [](int v, int count) { return v < count ? v : count - 1; };
  int start = 0, end = 0, shared = 0;
  if (l.num_groups > 0) {
    const int g = at_most(lane, l.num_groups);
    start = l.group_starts[g];
    end = l.group_starts[g + 1];
    shared = l.shared_lens[g];
  }
  int len = l.kv_lens[at_most(lane, l.num_seqs)];
  begins[lane] = 0;
  len = lane < l.num_seqs ? clamped(len, 0, l.most) : 0;
  start = clamped(start, 0, l.num_seqs);
  end = clamped(end, start, min(l.num_seqs, start + l.largest));
  shared = clamped(shared, 0, __shfl(len, start & 63, VELOX_WAVE));
  if (lane >= l.num_groups || end - start < 2) shared = 0;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (a wave's accesses to LDS are done in order)
  if (lane < l.num_groups && end > start) begins[start] = lane + 1;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  const int group = most_up_to_lane(begins[lane]) - 1;  // the last that begins at this lane's sequence or before, or -1
  const int its_end = __shfl(end, group & 63, VELOX_WAVE), its_shared = __shfl(shared, group & 63, VELOX_WAVE);
  const Own own = own_keys(group, group >= 0 && lane < its_end ? its_shared : 0, len);

  const int blocks = counts.blocks(l, end - start, shared), steps = counts.steps(shared), tiles = counts.tiles(own);
  auto sum = [](int v) { return __builtin_amdgcn_readlane(sum_up_to_lane(v), 63); };
  const int per = counts.fitted(l, counts.per(l, sum(blocks * steps), sum(counts.own_blocks * tiles)), [&](int p) { return sum(p > 0 ? blocks * parts_of(steps, p) : blocks); },
                                [&]() { return __builtin_amdgcn_readlane(most_up_to_lane(counts.most_parts(own)), 63); });
  const int items = blocks * parts_of(steps, per), upto = sum_up_to_lane(items), group_items = __builtin_amdgcn_readlane(upto, 63);
  auto of = [](int v, int at) { return __builtin_amdgcn_readlane(v, at); };
  if (wg < group_items) {
    const int at = __ffsll((unsigned long long)__ballot(upto > wg)) - 1, first = of(start, at);
    return counts.of_group(l, wg, wg - of(upto - items, at), at, first, of(end, at) - first, of(shared, at), per);
  }
  // every sequence has one item at least; its first one's wave writes down where its rows lie
  const int item = (wg - group_items) * WAVES + wave, parts = max(1, parts_of(tiles, per)), own_items = lane < l.num_seqs ? counts.own_blocks * parts : 0;
  const int own_upto = sum_up_to_lane(own_items);
  const uint64_t holds = __ballot(own_upto > item);
  if (holds == 0) return Item{-1, -1, 0, 0, 0, 0, 0, 0};
  const int at = __ffsll((unsigned long long)holds) - 1, first = of(own_upto - own_items, at), from = of(own.from, at), its_group = of(own.group, at);
  if (item == first && blockIdx.x == 0) {
    Directory rows = {0, 0, 0, (group_items << counts.block_shift) + first * 16, of(parts, at), {}};
    if (its_group >= 0) {
      rows.shared_at = (of(upto - items, its_group) << counts.block_shift) + (at - of(start, its_group)) * l.group;
      rows.shared_stride = of(blocks, its_group) << counts.block_shift;
      rows.shared_parts = parts_of(counts.steps(from), per);
    }
    if (lane == 0) directory[at] = rows;
  }
  return counts.of_sequence(item, item - first, at, from, of(own.to, at), per, group_items);
}

// With more of either a workgroup ahead works all items out (240 sequences 4.6 us, 1,000 6.5): a thread has a group and a sequence of its own (of these as many at a time), then every item is
// looked up by halving.  planned: [workgroup][wave], a group's item four times.
constexpr int PLAN_THREADS = 1024;
static_assert(MOST_GROUPS <= PLAN_THREADS, "a thread has a group");
__global__ void __launch_bounds__(PLAN_THREADS) shared_prefix_plan_kernel(const Lengths l, int tile_shift, int step_shift, int workgroups, Item* __restrict__ planned,
                                                                          Directory* __restrict__ directory) {
  __shared__ int lens[PLAN_THREADS], start[MOST_GROUPS], end[MOST_GROUPS], shared[MOST_GROUPS], before[MOST_GROUPS];
  __shared__ int upto[PLAN_THREADS], from[PLAN_THREADS], to[PLAN_THREADS];
  typedef int two_t __attribute__((ext_vector_type(2)));
  __shared__ two_t wave_sums[2][PLAN_THREADS / 64];
  __shared__ int most_of[PLAN_THREADS / 64];
  const Counts counts(l, tile_shift, step_shift);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, threads = blockDim.x;  // (as many as there are groups, at least)
  int turn = 0;
  struct Sums { int groups, own, all_groups, all_own; };  // up to this thread, and of all
  auto sums_up_to_thread = [&](int groups, int own) {
    const two_t in_wave = {sum_up_to_lane(groups), sum_up_to_lane(own)};
    turn ^= 1;
    if (lane == 63) wave_sums[turn][wave] = in_wave;
    __syncthreads();
    const two_t other = lane < threads / 64 ? wave_sums[turn][lane] : two_t{0, 0};
    const int others[2] = {sum_up_to_lane(other[0]), sum_up_to_lane(other[1])};
    const int before_wave = __builtin_amdgcn_readfirstlane(wave) - 1;
    Sums sums = {in_wave[0], in_wave[1], __builtin_amdgcn_readlane(others[0], 63), __builtin_amdgcn_readlane(others[1], 63)};
    if (before_wave >= 0) {
      sums.groups += __builtin_amdgcn_readlane(others[0], before_wave);
      sums.own += __builtin_amdgcn_readlane(others[1], before_wave);
    }
    return sums;
  };
  auto keys_of = [&](int b) { return clamped(l.kv_lens[b], 0, l.most); };
  int first = 0, behind = 0, keys = 0;
  if (tid < l.num_groups) {
    first = l.group_starts[tid];
    behind = l.group_starts[tid + 1];
    keys = l.shared_lens[tid];
  }
  const int len0 = tid < l.num_seqs ? keys_of(tid) : 0;
  lens[tid] = len0;
  __syncthreads();
  int steps = 0, blocks = 0;
  if (tid < l.num_groups) {
    first = clamped(first, 0, l.num_seqs);
    behind = clamped(behind, first, min(l.num_seqs, first + l.largest));
    keys = behind - first > 1 ? clamped(keys, 0, first < threads ? lens[first] : keys_of(first)) : 0;
    start[tid] = first;
    end[tid] = behind;
    shared[tid] = keys;
    steps = counts.steps(keys);
    blocks = counts.blocks(l, behind - first, keys);
  }
  __syncthreads();
  auto own_of = [&](int b, int keys) {
    int lo = -1, hi = l.num_groups;  // the last group that begins at b or before
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (start[mid] <= b) lo = mid;
      else hi = mid;
    }
    return own_keys(lo, lo >= 0 && b < end[lo] ? shared[lo] : 0, keys);
  };
  Own own = tid < l.num_seqs ? own_of(tid, len0) : Own{-1, 0, 0};
  int tiles = counts.tiles(own), most_parts = counts.most_parts(own);
  for (int b = threads + tid; b < l.num_seqs; b += threads) {
    const Own other = own_of(b, keys_of(b));
    tiles += counts.tiles(other);
    most_parts = max(most_parts, counts.most_parts(other));
  }
  const Sums work = sums_up_to_thread(blocks * steps, counts.own_blocks * tiles);
  const int per = counts.fitted(l, counts.per(l, work.all_groups, work.all_own), [&](int p) { return sums_up_to_thread(p > 0 ? blocks * parts_of(steps, p) : blocks, 0).all_groups; },
                                [&]() {
                                  const int in_wave = __builtin_amdgcn_readlane(most_up_to_lane(most_parts), 63);
                                  if (lane == 0) most_of[wave] = in_wave;
                                  __syncthreads();
                                  return __builtin_amdgcn_readlane(most_up_to_lane(lane < threads / 64 ? most_of[lane] : 0), 63);
                                });
  const int items = blocks * parts_of(steps, per);
  int group_items = 0, own_items = 0;
  for (int base = 0; base < l.num_seqs; base += threads) {
    const int b = base + tid;
    if (base > 0) own = b < l.num_seqs ? own_of(b, keys_of(b)) : Own{-1, 0, 0};
    const int parts = max(1, parts_of(counts.tiles(own), per)), its_items = b < l.num_seqs ? counts.own_blocks * parts : 0;
    const Sums sums = sums_up_to_thread(items, its_items);  // (its barrier: everybody is done with what the sequences before have left here)
    group_items = sums.all_groups;
    if (base == 0 && tid < l.num_groups) before[tid] = sums.groups - items;
    upto[tid] = sums.own;
    from[tid] = own.from;
    to[tid] = own.to;
    __syncthreads();
    if (b < l.num_seqs) {
      Directory rows = {0, 0, 0, (group_items << counts.block_shift) + (own_items + sums.own - its_items) * 16, parts, {}};
      if (own.group >= 0) {
        rows.shared_at = (before[own.group] << counts.block_shift) + (b - start[own.group]) * l.group;
        rows.shared_stride = counts.blocks(l, end[own.group] - start[own.group], shared[own.group]) << counts.block_shift;
        rows.shared_parts = parts_of(counts.steps(own.from), per);
      }
      directory[b] = rows;
    }
    for (int t = tid; t < sums.all_own; t += threads) {
      int lo = -1, hi = threads - 1;  // the first sequence that has an item behind t
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (upto[mid] > t) hi = mid;
        else lo = mid;
      }
      const int item = own_items + t, record = min(group_items, workgroups) * WAVES + item;  // (groups that overlap may have more)
      if (record < workgroups * WAVES) planned[record] = counts.of_sequence(item, t - (hi > 0 ? upto[hi - 1] : 0), base + hi, from[hi], to[hi], per, group_items);
    }
    own_items += sums.all_own;
  }
  const int group_records = min(group_items, workgroups) * WAVES;
  for (int record = tid; record < group_records; record += threads) {
    const int item = record / WAVES;
    int lo = 0, hi = l.num_groups;  // the last group with no more items before it (one without items has as many as the next)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (before[mid] <= item) lo = mid;
      else hi = mid;
    }
    planned[record] = counts.of_group(l, item, item - before[lo], lo, start[lo], end[lo] - start[lo], shared[lo], per);
  }
  for (int record = group_records + own_items + tid; record < workgroups * WAVES; record += threads) planned[record] = Item{-1, -1, 0, 0, 0, 0, 0, 0};
}

// ---- rows against a stream of keys ----------------------------------------------------------------------------------------
template <typename T> struct Cache {
  const T* k;
  const T* v;
  int nkv, page_shift;
  uint32_t last_page;  // (an id beyond it, which no table should hold, reads this one)
};

template <typename T, int RT> struct Rows {  // RT tiles of 16 rows, in a wave
  static constexpr int NQB = (D + Block<T>::KB - 1) / Block<T>::KB;  // contraction blocks of K Q^T (beyond the head size: zeros)
  static constexpr int NC = D / 16;
  float4_t q[RT][NQB], acc[RT][NC];
  float m[RT], l[RT];  // the running maximum, and this lane's keys' part of the sum
};

// query(r): the address of row r's query, or nullptr
template <typename T, int RT, typename QueryOf> __device__ __forceinline__ void begin_rows(Rows<T, RT>& rows, QueryOf query) {
  typedef Block<T> B;
  const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const T* q = query(16 * rt + i);
#pragma unroll
    for (int cb = 0; cb < Rows<T, RT>::NQB; ++cb) {
      rows.q[rt][cb] = float4_t{0.f, 0.f, 0.f, 0.f};
      if (q != nullptr && (D % B::KB == 0 || B::KB * cb + B::VEC * g < D)) rows.q[rt][cb] = *reinterpret_cast<const float4_t*>(q + B::KB * cb + B::VEC * g);
    }
    rows.m[rt] = -INFINITY;
    rows.l[rt] = 0.f;
#pragma unroll
    for (int c = 0; c < Rows<T, RT>::NC; ++c) rows.acc[rt][c] = float4_t{0.f, 0.f, 0.f, 0.f};
  }
}

// The rows against those of the keys [lo, hi) of a table's sequence that lie in tiles first, first + stride, ...
template <typename T, int RT>
__device__ __forceinline__ void stream_keys(Rows<T, RT>& rows, const Cache<T>& cache, int kvh, const int* __restrict__ table, int lo, int hi, int first, int stride, float scale) {
  typedef Block<T> B;
  constexpr int KB = B::KB, VEC = B::VEC, NQB = Rows<T, RT>::NQB, NC = Rows<T, RT>::NC;
  constexpr int TILE = KB, NU = KB / 16;
  const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
  const int page_size = 1 << cache.page_shift;
  const int end = (hi + TILE - 1) / TILE;
  if (first >= end) return;
  const int last = first + (end - 1 - first) / stride * stride;

  // Keys beyond either end are read from the nearest place inside: their scores are masked and their values zeroed.  (A lane's keys of both
  // score tiles lie in one run of eight in bfloat16, and so in one page.)
  auto key_at = [&](int tile, int u) { return clamped(TILE * tile + B::key_row(u, i), lo, hi - 1); };
  auto value_at = [&](int tile) { return clamped(TILE * tile + VEC * g, lo & ~(VEC - 1), (hi - 1) & ~(VEC - 1)); };
  struct Ids { uint32_t k[NU], v; };
  auto load_ids = [&](int tile) {
    Ids ids;
#pragma unroll
    for (int u = 0; u < NU; ++u) ids.k[u] = min((uint32_t)table[key_at(tile, u) >> cache.page_shift], cache.last_page);
    ids.v = min((uint32_t)table[value_at(tile) >> cache.page_shift], cache.last_page);
    return ids;
  };
  float4_t k[NU][NQB], v[NC];
  auto load_keys = [&](const Ids& ids, int tile) {
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int n = key_at(tile, u);
      const T* p = cache.k + ((((size_t)ids.k[u] * cache.nkv + kvh) << cache.page_shift) + (n & (page_size - 1))) * D + VEC * g;
#pragma unroll
      for (int cb = 0; cb < NQB; ++cb) {
        // (of a block that reaches beyond the head size, lanes there read the row's beginning and hold zeros)
        const bool inside = D % KB == 0 || KB * cb + VEC * g < D;
        k[u][cb] = *reinterpret_cast<const float4_t*>(p + (inside ? KB * cb : -VEC * g));
        if (!inside) k[u][cb] = float4_t{0.f, 0.f, 0.f, 0.f};
      }
    }
  };
  auto load_values = [&](const Ids& ids, int tile) {
    const int n = value_at(tile);
    const T* p = cache.v + ((((size_t)ids.v * cache.nkv + kvh) * D + i) << cache.page_shift) + (n & (page_size - 1));
#pragma unroll
    for (int c = 0; c < NC; ++c) v[c] = *reinterpret_cast<const float4_t*>(p + ((size_t)(16 * c) << cache.page_shift));
  };
  const float scale_eff = scale * B::SCALE;

  Ids ids = load_ids(first), next_ids = load_ids(min(first + stride, last));
  load_keys(ids, first);
  load_values(ids, first);
  for (int tile = first; tile < end; tile += stride) {
    const int n0 = TILE * tile, next = min(tile + stride, last);  // (what is asked for behind the last tile is the last tile again)
    const bool whole = n0 >= lo && n0 + TILE <= hi;               // (the same for the whole wave)
    float4_t s[RT][NU];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        s[rt][u] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int cb = 0; cb < NQB; ++cb) s[rt][u] = B::mma(k[u][cb], rows.q[rt][cb], s[rt][u]);
      }
    ids = next_ids;
    next_ids = load_ids(min(tile + 2 * stride, last));
    load_keys(ids, next);
    float4_t pf[RT];
    float alpha[RT];
    bool moved = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      if (!whole) {
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int n = n0 + B::first_score(u, g) + j;
            s[rt][u][j] = n >= lo && n < hi ? s[rt][u][j] : -INFINITY;
          }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = fmaxf(mx, s[rt][u][j]);
      mx = fmaxf(mx, __shfl_xor(mx, 16, VELOX_WAVE));
      mx = fmaxf(mx, __shfl_xor(mx, 32, VELOX_WAVE));
      // What a row's exponents refer to need not be its maximum: it is moved, and all that was gathered rescaled, only when a score lies more than
      // SLACK above it (bfloat16; in powers of two: weights stay below 2^8, and are rounded relative to themselves).
      constexpr float SLACK = sizeof(T) == 2 ? 8.f : 0.f;
      const float top = mx * scale_eff;  // (the scale is positive)
      const bool stays = top - rows.m[rt] <= SLACK;  // (false while the row has seen no key: -inf)
      const float m_new = stays ? rows.m[rt] : fmaxf(rows.m[rt], top);
      const float m_safe = m_new == -INFINITY ? 0.f : m_new;
      alpha[rt] = stays ? 1.f : rows.m[rt] == -INFINITY ? 0.f : B::exp_of(rows.m[rt] - m_safe);
      moved = moved || !stays;
      float sum = 0.f;
      float p[NU][4];
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          p[u][j] = B::exp_of(fmaf(s[rt][u][j], scale_eff, -m_safe));
          sum += p[u][j];
        }
      if constexpr (sizeof(T) == 2) {
        bf16x8_t e;
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j) e[4 * u + j] = (bf16_t)p[u][j];  // weights are rounded to the values' type for the product
        pf[rt] = __builtin_bit_cast(float4_t, e);
      } else {
        pf[rt] = float4_t{p[0][0], p[0][1], p[0][2], p[0][3]};
      }
      rows.l[rt] = rows.l[rt] * alpha[rt] + sum;
      rows.m[rt] = m_new;
    }
    if (__ballot(moved) != 0ull) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int c = 0; c < NC; ++c) rows.acc[rt][c] = rows.acc[rt][c] * alpha[rt];
    }
    if (!whole) {
      const int n = n0 + VEC * g;
#pragma unroll
      for (int c = 0; c < NC; ++c) B::mask(v[c], lo - n, hi - n);
    }
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) rows.acc[rt][c] = B::mma(v[c], pf[rt], rows.acc[rt][c]);
    load_values(ids, next);
  }
}

template <typename T, int RT> __device__ __forceinline__ void finish_sums(Rows<T, RT>& rows) {
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    rows.l[rt] += __shfl_xor(rows.l[rt], 16, VELOX_WAVE);
    rows.l[rt] += __shfl_xor(rows.l[rt], 32, VELOX_WAVE);
  }
}

// The four waves' results of the same rows, put together a row tile at a time.  `scaled(row, top, total)`: what its sums of weighted values are multiplied by,
// given the exponents' reference (natural units) and the sum of weights; `leave(row, channel, four)`.
template <int RT> constexpr int join_bytes() { return WAVES * (D / 16) * 64 * 16 + 2 * WAVES * 16 * RT * 4; }
template <typename T, int RT, typename Scaled, typename Leave>
__device__ __forceinline__ void join_waves(Rows<T, RT>& rows, int count, char* smem, Scaled scaled, Leave leave) {
  typedef Block<T> B;
  constexpr int NC = D / 16;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, i = lane & 15;
  float4_t* const acc_all = reinterpret_cast<float4_t*>(smem);                 // [wave][channel tile][lane]
  float* const m_all = reinterpret_cast<float*>(smem + WAVES * NC * 64 * 16);  // [wave][16 RT]
  float* const l_all = m_all + WAVES * 16 * RT;
  finish_sums<T, RT>(rows);
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    if (g == 0) {
      m_all[wave * 16 * RT + 16 * rt + i] = rows.m[rt];
      l_all[wave * 16 * RT + 16 * rt + i] = rows.l[rt];
    }
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    if (rt > 0) __syncthreads();
#pragma unroll
    for (int c = 0; c < NC; ++c) acc_all[(wave * NC + c) * 64 + lane] = rows.acc[rt][c];
    __syncthreads();
    float top = -INFINITY, total = 0.f, weight[WAVES];
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, m_all[w * 16 * RT + 16 * rt + i]);
    const float safe = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float m = m_all[w * 16 * RT + 16 * rt + i];
      weight[w] = m == -INFINITY ? 0.f : B::exp_of(m - safe);
      total += weight[w] * l_all[w * 16 * RT + 16 * rt + i];
    }
    const bool there = 16 * rt + i < count;
    const float by = there ? scaled(16 * rt + i, top * B::LN_UNIT, total) : 0.f;
    for (int c = wave; c < NC; c += WAVES) {
      float4_t sum = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < WAVES; ++w) sum += acc_all[(w * NC + c) * 64 + lane] * weight[w];
      if (there) leave(16 * rt + i, 16 * c + 4 * g, sum * by);
    }
  }
}

// ---- many rows: tiles in LDS ------------------------------------------------------------------------------------------------------
// `idle`: the wave has no rows and only brings tiles.
// From some hundred rows on the products count, and every 32 rows reading the keys for themselves is more than the second-level caches give (448 rows behind 32,768 keys, 28
// heads over 4: 111 us that way, 65 this way).  Here the four
// waves have 32 rows each and share tiles of 64 keys (bfloat16, heads of 64 and 128 channels).  Every lane asks for 16 bytes of the cache with a
// load that writes LDS itself, a whole tile ahead of the one being multiplied, into the other of two buffers; one barrier a tile is left.  Such a load fills
// a contiguous kilobyte, so what lies where is decided by which piece each lane asks for: pieces of 16 bytes change places within a
// row such that eight lanes that read together touch eight different ones.  Piece c of key k lies at c ^ ((k & 3) | (k >> 3 & 1) << 2), piece c of channel d
// of V^T, whose rows are the tile's 64 keys, at c ^ (d & 7).
constexpr int TALL_TILE = 64, TALL_ROWS = 32 * WAVES;
constexpr bool HAS_TALL = D == 64 || D == 128;
constexpr int TALL_BYTES = TALL_TILE * D * 2;  // of the keys or the values of a tile
__device__ __forceinline__ void tall_item(Rows<bf16_t, 2>& rows, const Cache<bf16_t>& cache, int kvh, const int* __restrict__ table, int lo, int hi, float scale, bool idle,
                                          char (*smem)[2 * TALL_BYTES]) {
  typedef Block<bf16_t> B;
  constexpr int CT = 2, NQB = Rows<bf16_t, 2>::NQB, NC = D / 16, NT = TALL_TILE / 16, NKB = TALL_TILE / 32;
  constexpr int PIECES = D / 8;                  // of a key's row
  constexpr int LOADS = TALL_BYTES / 1024 / WAVES;  // of a wave, for the keys of a tile, and as many for the values
  constexpr int KEYS = 64 / PIECES;              // of one load
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, i = lane & 15;
  const int page_size = 1 << cache.page_shift;
  // what each lane asks for: of keys KEYS (wave + 4 m) + lane / PIECES, of channels 8 (wave + 4 m) + lane / 8
  const int key_in_load = lane / PIECES, first_key = KEYS * wave + key_in_load;
  const uint32_t key_bytes = (uint32_t)(key_in_load * D + 8 * ((lane % PIECES) ^ ((first_key & 3) | ((first_key >> 3) & 1) << 2))) * 2;
  const int value_eight = (lane & 7) ^ ((lane >> 3) & 7);  // which eight of the tile's keys
  const size_t page_elems = ((size_t)cache.nkv * D) << cache.page_shift;
  const size_t value_elems = (size_t)(kvh * D + 8 * wave + (lane >> 3)) << cache.page_shift;
  // lane e's page id, e < 8, is that of the tile's keys 8 e .. 8 e + 7, or of the last keys there are
  auto load_id = [&](int n0) { return min((uint32_t)table[min(n0 + 8 * (lane & 7), hi - 1) >> cache.page_shift], cache.last_page); };
  auto issue_keys = [&](int n0, uint32_t id, int buffer) {
    const int at = __builtin_amdgcn_readfirstlane(n0);
    char* const to = smem[__builtin_amdgcn_readfirstlane(buffer)];
#pragma unroll
    for (int m = 0; m < LOADS; ++m) {
      const int key0 = KEYS * (wave + WAVES * m);
      const size_t page = (size_t)(uint32_t)__builtin_amdgcn_readlane(id, key0 >> 3);
      const bf16_t* base = cache.k + (((page * cache.nkv + kvh) << cache.page_shift) + ((at + key0) & (page_size - 1))) * D;
      load_to_lds_16(base, key_bytes, to + 1024 * (wave + WAVES * m));
    }
  };
  auto issue_values = [&](int n0, uint32_t id, int buffer) {
    const int at = __builtin_amdgcn_readfirstlane(n0);
    char* const to = smem[__builtin_amdgcn_readfirstlane(buffer)] + TALL_BYTES;
    const uint32_t page = __shfl(id, value_eight, VELOX_WAVE);
    const bf16_t* from = cache.v + (size_t)page * page_elems + (value_elems + (uint32_t)((at + 8 * value_eight) & (page_size - 1)));
#pragma unroll
    for (int m = 0; m < LOADS; ++m) load_to_lds_16(from + ((size_t)(8 * WAVES * m) << cache.page_shift), to + 1024 * (wave + WAVES * m));
  };
  // where each lane reads its operands: row 8 (i / 4) + i % 4 of a block of 32 keys (+ 4 u for score tile u), pieces 4 cb + g; row i of a channel tile,
  // pieces 4 kb + g
  const int half = (i >> 2) & 1;
  const int key_row = (8 * (i >> 2) + (i & 3)) * (2 * D) + 16 * (g ^ (i & 3)), value_row = TALL_BYTES + i * 128 + 16 * (g ^ (i & 3));
  const int key_even = key_row + 64 * half, key_odd = key_row + 64 * (1 - half);
  const int value_first = value_row + 64 * half, value_second = value_row + 64 * (1 - half);
  const float scale_eff = scale * B::SCALE;

  // Operands are read a few products ahead, in this order: left to the compiler, which has no registers to spare here, most were read right before their
  // product, and its wait was longer than the product (one group behind 32,768 keys 86 us, this way 82).
  constexpr int KEYS_AHEAD = 6, VALUES_AHEAD = 3;
  auto multiply_keys = [&](float4_t (&s)[CT][NT], const char* tile) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) s[ct][t] = float4_t{0.f, 0.f, 0.f, 0.f};
    float4_t k[KEYS_AHEAD];
    auto read = [&](int e) {  // contraction block e % NQB of score tile e / NQB
      const int t = e / NQB, cb = e % NQB;
      k[e % KEYS_AHEAD] = *reinterpret_cast<const float4_t*>(tile + ((cb & 1) ? key_odd : key_even) + 128 * (cb >> 1) + (32 * (t >> 1) + 4 * (t & 1)) * (2 * D));
    };
#pragma unroll
    for (int e = 0; e < KEYS_AHEAD - 1; ++e) read(e);
#pragma unroll
    for (int e = 0; e < NT * NQB; ++e) {
      if (e + KEYS_AHEAD - 1 < NT * NQB) read(e + KEYS_AHEAD - 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) s[ct][e / NQB] = B::mma(k[e % KEYS_AHEAD], rows.q[ct][e % NQB], s[ct][e / NQB]);
    }
  };
  // A tile's keys are asked for two tiles ahead of its values' product and its values one: while the weights of a tile are worked out from their
  // scores, the next tile's scores are already being multiplied.
  uint32_t id = load_id(lo), next_id = load_id(lo + TALL_TILE), far_id = load_id(lo + 2 * TALL_TILE);
  __builtin_amdgcn_s_waitcnt(0x0F70);  // (the queries have arrived, said in a way the compiler sees: it would otherwise wait in every round)
  issue_keys(lo, id, 0);
  wait_for_loads<0>();
  __syncthreads();
  issue_values(lo, id, 0);
  if (lo + TALL_TILE < hi) issue_keys(lo + TALL_TILE, next_id, 1);
  float4_t s0[CT][NT], s1[CT][NT];
  if (!idle) multiply_keys(s0, smem[0]);
  auto round = [&](float4_t (&s)[CT][NT], float4_t (&next)[CT][NT], int n0, int buffer) {
    wait_for_loads<0>();  // this wave's pieces of this tile's values and the next one's keys have landed
    __syncthreads();      // everybody's have, and everybody is done with the buffers that are filled now
    id = next_id;
    next_id = far_id;
    far_id = load_id(n0 + 3 * TALL_TILE);
    if (n0 + TALL_TILE < hi) issue_values(n0 + TALL_TILE, id, buffer ^ 1);
    if (n0 + 2 * TALL_TILE < hi) issue_keys(n0 + 2 * TALL_TILE, next_id, buffer);
    if (idle) return;
    const bool whole = n0 + TALL_TILE <= hi;
    if (!whole) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[ct][t][j] = n0 + 32 * (t >> 1) + 8 * g + 4 * (t & 1) + j < hi ? s[ct][t][j] : -INFINITY;
    }
    // (matrix instructions first: the other wave of the SIMD then has the vector unit for its weights meanwhile)
    __builtin_amdgcn_s_setprio(1);
    multiply_keys(next, smem[buffer ^ 1]);  // (behind the last tile: of whatever lies there, and not used)
    __builtin_amdgcn_s_setprio(0);
    float alpha[CT];
    float4_t pf[CT][NKB];
    bool moved = false;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      float mx = -INFINITY;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = fmaxf(mx, s[ct][t][j]);
      mx = fmaxf(mx, __shfl_xor(mx, 16, VELOX_WAVE));
      mx = fmaxf(mx, __shfl_xor(mx, 32, VELOX_WAVE));
      const float top = mx * scale_eff;
      const bool stays = top - rows.m[ct] <= 8.f;  // (see stream_keys)
      const float m_new = stays ? rows.m[ct] : fmaxf(rows.m[ct], top);
      const float m_safe = m_new == -INFINITY ? 0.f : m_new;
      alpha[ct] = stays ? 1.f : rows.m[ct] == -INFINITY ? 0.f : B::exp_of(rows.m[ct] - m_safe);
      moved = moved || !stays;
      float sum = 0.f;
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) {
        bf16x8_t e;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float p = B::exp_of(fmaf(s[ct][2 * kb + u][j], scale_eff, -m_safe));
            sum += p;
            e[4 * u + j] = (bf16_t)p;
          }
        pf[ct][kb] = __builtin_bit_cast(float4_t, e);
      }
      rows.l[ct] = rows.l[ct] * alpha[ct] + sum;
      rows.m[ct] = m_new;
    }
    if (__ballot(moved) != 0ull) {
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) rows.acc[ct][c] = rows.acc[ct][c] * alpha[ct];
    }
    char* const tile = smem[buffer];
    if (!whole) {
      // Values behind the last key become zeros where they lie (every wave does it for itself, all to the same): asked for in the loop below, every
      // channel tile would wait for its values on its own.
#pragma unroll 1
      for (int p = lane; p < 8 * D; p += 64) {
        float4_t* const at = reinterpret_cast<float4_t*>(tile + TALL_BYTES + (p >> 3) * 128 + 16 * ((p & 7) ^ ((p >> 3) & 7)));
        float4_t v = *at;
        B::mask(v, 0, hi - (n0 + 8 * (p & 7)));
        *at = v;
      }
    }
    __builtin_amdgcn_s_setprio(1);
    float4_t v[VALUES_AHEAD][NKB];
    auto read = [&](int c) {
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) v[c % VALUES_AHEAD][kb] = *reinterpret_cast<const float4_t*>(tile + (kb ? value_second : value_first) + 2048 * c);
    };
#pragma unroll
    for (int c = 0; c < VALUES_AHEAD - 1; ++c) read(c);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (c + VALUES_AHEAD - 1 < NC) read(c + VALUES_AHEAD - 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) rows.acc[ct][c] = B::mma(v[c % VALUES_AHEAD][kb], pf[ct][kb], rows.acc[ct][c]);
    }
    __builtin_amdgcn_s_setprio(0);
  };
  for (int n0 = lo; n0 < hi; n0 += 2 * TALL_TILE) {
    round(s0, s1, n0, 0);
    if (n0 + TALL_TILE < hi) round(s1, s0, n0 + TALL_TILE, 1);
  }
}

// A wave's rows, put where the joining kernel finds them.
template <typename T, int RT> __device__ __forceinline__ void leave_rows(Rows<T, RT>& rows, int count, float* __restrict__ part_o, float* __restrict__ part_lse) {
  const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
  finish_sums<T, RT>(rows);
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    if (16 * rt + i >= count) continue;
    const float inv = rows.l[rt] > 0.f ? 1.f / rows.l[rt] : 1.f;
    float* const to = part_o + (size_t)(16 * rt + i) * D + 4 * g;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) *reinterpret_cast<float4_t*>(to + 16 * c) = rows.acc[rt][c] * inv;
    if (g == 0) part_lse[16 * rt + i] = rows.l[rt] > 0.f ? rows.m[rt] * Block<T>::LN_UNIT + logf(rows.l[rt]) : -INFINITY;
  }
}

// Two workgroups to a compute unit where a wave's registers allow it.
constexpr int workgroups_per_unit() { return D <= 128 ? 2 : 1; }

// part_o: [KV head][rows_room][D], part_lse: [KV head][rows_room]; directory: [sequence]
// RT = TALL: rows in blocks of TALL_ROWS over tiles in LDS.
constexpr int TALL = TALL_ROWS / 16;
template <typename T> constexpr int tile_shift() { return sizeof(T) == 2 ? 5 : 4; }
template <typename T, int RT> constexpr int step_shift() { return RT == TALL ? 6 : tile_shift<T>() + 2; }
template <typename T, int RT>
__global__ void __launch_bounds__(THREADS, (RT == TALL ? 2 : workgroups_per_unit()))
shared_prefix_kernel(const T* __restrict__ qkv, int qkv_stride, const Cache<T> cache, const int* __restrict__ block_tables, int table_width, const Lengths l, float scale,
                     float* __restrict__ part_o, float* __restrict__ part_lse, Directory* __restrict__ directory) {
  constexpr int TILE = Block<T>::KB, R = 16 * RT;
  __shared__ __attribute__((aligned(1024))) char smem[RT == TALL ? 4 * TALL_BYTES : join_bytes<RT>()];
  __shared__ int begins[THREADS];
  const int kvh = blockIdx.x, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Item item;
  if (l.planned != nullptr) {
    const Item planned = l.planned[blockIdx.y * WAVES + wave];
    auto of = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    item = Item{of(planned.group), of(planned.sequence), of(planned.first), of(planned.count), of(planned.block), of(planned.from), of(planned.to), of(planned.at)};
  } else {
    item = find_item(l, Counts(l, tile_shift<T>(), step_shift<T, RT>()), blockIdx.y, begins + 64 * wave, directory);
  }
  const int heads = l.group;
  float* const o = part_o + (size_t)kvh * l.rows_room * D;
  float* const lse = part_lse + (size_t)kvh * l.rows_room;
  if (item.group >= 0) {
    if (item.at < 0 || item.at + R > l.rows_room) return;  // (groups that overlap: no more than there is room for)
    const int first_row = item.block * R, rows_all = item.count * heads;
    const int* const table = block_tables + (size_t)item.first * table_width;
    auto query_of = [&](int row) -> const T* {
      return row < rows_all ? qkv + (size_t)(item.first + row / heads) * qkv_stride + (size_t)(kvh * heads + row % heads) * D : nullptr;
    };
    if constexpr (RT == TALL) {
      const int wave_row = 32 * wave;
      Rows<T, 2> rows;
      begin_rows<T, 2>(rows, [&](int r) { return query_of(first_row + wave_row + r); });
      tall_item(rows, cache, kvh, table, item.from, item.to, scale, first_row + wave_row >= rows_all, reinterpret_cast<char(*)[2 * TALL_BYTES]>(smem));
      leave_rows<T, 2>(rows, rows_all - first_row - wave_row, o + (size_t)(item.at + wave_row) * D, lse + item.at + wave_row);
    } else {
      Rows<T, RT> rows;
      begin_rows<T, RT>(rows, [&](int r) { return query_of(first_row + r); });
      stream_keys<T, RT>(rows, cache, kvh, table, item.from, item.to, item.from / TILE + wave, WAVES, scale);
      join_waves<T, RT>(rows, rows_all - first_row, smem,
                        [&](int row, float top, float total) {
                          if (wave == 0 && lane < 16) lse[item.at + row] = total > 0.f ? top + logf(total) : -INFINITY;
                          return total > 0.f ? 1.f / total : 1.f;
                        },
                        [&](int row, int channel, const float4_t& four) { *reinterpret_cast<float4_t*>(o + (size_t)(item.at + row) * D + channel) = four; });
    }
    return;
  }
  if (item.sequence < 0 || item.at < 0 || item.at + 16 > l.rows_room) return;
  Rows<T, 1> rows;
  begin_rows<T, 1>(rows, [&](int r) -> const T* {
    const int row = item.block * 16 + r;
    return row < heads ? qkv + (size_t)item.sequence * qkv_stride + (size_t)(kvh * heads + row) * D : nullptr;
  });
  if (item.to > item.from)
    stream_keys<T, 1>(rows, cache, kvh, block_tables + (size_t)item.sequence * table_width, item.from, item.to, item.from / TILE, 1, scale);
  leave_rows<T, 1>(rows, heads - 16 * item.block, o + (size_t)item.at * D, lse + item.at);
}

// Few keys: a workgroup per (KV head, sequence, 16 of its rows) takes all of them, the shared ones too, and leaves the result itself: no plan, no parts, nothing to
// join.  What bounds it is latency: a launch (1.6 us), lengths, page ids and keys that wait for one another (0.8 us each), then about 0.7 us for each of a
// wave's tiles; 4 sequences of 321 keys (12 heads over 2) take 8.3 us (traced).  (With how many keys sharing them out is better: see the host's rule.)
template <typename T>
__global__ void __launch_bounds__(THREADS, workgroups_per_unit())
shared_prefix_direct_kernel(const T* __restrict__ qkv, int qkv_stride, const Cache<T> cache, const int* __restrict__ block_tables, int table_width, const Lengths l, float scale,
                            const float* __restrict__ sinks, T* __restrict__ out) {
  constexpr int TILE = Block<T>::KB;
  __shared__ __attribute__((aligned(16))) char smem[join_bytes<1>()];
  const int kvh = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int heads = l.group, first_row = 16 * blockIdx.z, len = clamped(l.kv_lens[b], 0, l.most);
  int first = b, shared = 0;
  for (int base = 0; base < l.num_groups; base += 64) {
    const int g = min(base + lane, l.num_groups - 1);
    const int start = clamped(l.group_starts[g], 0, l.num_seqs), end = clamped(l.group_starts[g + 1], start, min(l.num_seqs, start + l.largest)), keys = l.shared_lens[g];
    const uint64_t holds = __ballot(base + lane < l.num_groups && start <= b && b < end && end - start > 1);
    if (holds != 0) {
      const int at = 63 - __builtin_clzll(holds);
      first = __builtin_amdgcn_readlane(start, at);
      shared = __builtin_amdgcn_readlane(keys, at);
    }
  }
  shared = clamped(shared, 0, first == b ? len : clamped(l.kv_lens[first], 0, l.most));
  if (shared > len) shared = 0;
  Rows<T, 1> rows;
  begin_rows<T, 1>(rows, [&](int r) -> const T* {
    return first_row + r < heads ? qkv + (size_t)b * qkv_stride + (size_t)(kvh * heads + first_row + r) * D : nullptr;
  });
  // (a sequence's own tiles begin with the wave that the shared ones end before)
  const int shared_tiles = (shared + TILE - 1) / TILE;
  if (shared > 0) stream_keys<T, 1>(rows, cache, kvh, block_tables + (size_t)first * table_width, 0, shared, wave, WAVES, scale);
  if (len > shared)
    stream_keys<T, 1>(rows, cache, kvh, block_tables + (size_t)b * table_width, shared, len, shared / TILE + ((wave - shared_tiles) & (WAVES - 1)), WAVES, scale);
  T* const to = out + ((size_t)b * l.group * cache.nkv + kvh * heads + first_row) * D;
  join_waves<T, 1>(rows, heads - first_row, smem,
                   [&](int row, float top, float total) {
                     if (total <= 0.f) return 1.f;
                     return 1.f / (total + (sinks != nullptr ? expf(sinks[kvh * heads + first_row + row] - top) : 0.f));
                   },
                   [&](int row, int channel, const float4_t& four) {
                     T* const dst = to + (size_t)row * D + channel;
#pragma unroll
                     for (int j = 0; j < 4; ++j) dst[j] = from_f32<T>(four[j]);
                   });
}

// A wave per (head, sequence): the parts that hold its row, joined.  Lane p asks for part p's log-sum (the next 64 parts', if there are more, in
// another round) and every lane for its own channels of up to JOINED_AT_ONCE parts, all before it waits for any of them.  A sink adds exp(sink) to the
// denominator.  (About 4 us for small calls: a launch and three loads in a row; 64 sequences of 28 heads with 27 parts 6.5 us, 24 MB at 3.7 TB/s.)
constexpr int JOIN_HEADS = 4;
template <typename T>
__global__ void __launch_bounds__(64 * JOIN_HEADS) shared_prefix_join_kernel(int nh, int group, int rows_room, const Directory* __restrict__ directory,
                                                                             const float* __restrict__ part_o, const float* __restrict__ part_lse,
                                                                             const float* __restrict__ sinks, T* __restrict__ out) {
  typedef float channels_t __attribute__((ext_vector_type(LANE_CHANNELS)));
  const int lane = threadIdx.x & 63, head = blockIdx.x * JOIN_HEADS + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), b = blockIdx.y;
  if (head >= nh) return;
  const Directory d = directory[b];
  const int kvh = head / group, h = head - kvh * group, own_stride = (group + 15) / 16 * 16;
  const int shared_parts = clamped(d.shared_parts, 0, rows_room / 16), parts = shared_parts + clamped(d.own_parts, 0, rows_room / 16);  // (of groups that overlap nobody
  auto place_of = [&](int part) -> size_t {                                                                                             // may have written it down)
    const unsigned row = part < shared_parts ? (unsigned)d.shared_at + (unsigned)part * (unsigned)d.shared_stride
                                             : (unsigned)d.own_at + (unsigned)(part - shared_parts) * (unsigned)own_stride;
    return (size_t)kvh * rows_room + min(row + (unsigned)h, (unsigned)rows_room - 1u);
  };
  const bool live = lane * LANE_CHANNELS < D;
  const float* const channels = part_o + (live ? lane * LANE_CHANNELS : 0);
  float top = -INFINITY, denom = 0.f;
  channels_t acc = 0.f;
  for (int p0 = 0; p0 < parts; p0 += 64) {
    const int here = min(parts - p0, 64);
    const float log_sum = lane < here ? part_lse[place_of(p0 + lane)] : -INFINITY;
    auto join = [&](auto ahead) {
      constexpr int N = decltype(ahead)::value;
      channels_t o[N];
#pragma unroll
      for (int j = 0; j < N; ++j)
        o[j] = *reinterpret_cast<const channels_t*>(channels + place_of(p0 + (j < here ? j : here - 1)) * D);  // (no branch, or each would wait for the one before)
      const float now = fmaxf(top, wave_max(log_sum)), safe = now == -INFINITY ? 0.f : now, old = top == -INFINITY ? 0.f : expf(top - safe);
      const float weight = log_sum == -INFINITY ? 0.f : expf(log_sum - safe);
      denom = denom * old + wave_sum(weight);
      acc = acc * old;
      top = now;
      auto weight_of = [&](int j) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(weight), j)); };
#pragma unroll
      for (int j = 0; j < N; ++j) acc += (j < here ? o[j] : channels_t(0.f)) * weight_of(j);  // (a part without a key holds zeros)
      for (int j = N; j < here; ++j) acc += *reinterpret_cast<const channels_t*>(channels + place_of(p0 + j) * D) * weight_of(j);
    };
    if (here <= 6) join(std::integral_constant<int, 6>{});
    else join(std::integral_constant<int, JOINED_AT_ONCE>{});
  }
  if (sinks != nullptr && top != -INFINITY) denom += expf(sinks[head] - top);
  if (!live) return;
  acc = acc * (denom > 0.f ? 1.f / denom : 1.f);
  T* const dst = out + ((size_t)b * nh + head) * D + lane * LANE_CHANNELS;
#pragma unroll
  for (int j = 0; j < LANE_CHANNELS; ++j) dst[j] = from_f32<T>(acc[j]);
}

// Row tiles a wave can hold: its registers hold the queries, the output and a tile of keys and values.  (In float32 two never pay over more workgroups of one: see the
// host's rule.)
template <typename T> constexpr int most_row_tiles() { return sizeof(T) == 2 && D <= 128 ? 2 : 1; }

extern "C" int velox_shared_prefix_head_dim() { return D; }
extern "C" int velox_shared_prefix_most_groups() { return MOST_GROUPS; }
extern "C" int velox_shared_prefix_most_keys() { return MOST_KEYS; }
static bool has_row_tiles(int row_tiles, int dtype) {  // 0: all keys in one workgroup
  if (row_tiles < 0 || (row_tiles & (row_tiles - 1)) != 0) return false;
  return row_tiles <= (dtype == VELOX_BF16 ? most_row_tiles<bf16_t>() : most_row_tiles<float>()) || (row_tiles == TALL && dtype == VELOX_BF16 && HAS_TALL);
}

// items: workgroups per KV head, and rows_room: rows per KV head, at least what velox_shared_prefix_room gives.  part_o: float32 [nkv, rows_room, D],
// part_lse: float32 [nkv, rows_room], directory: eight int32 a sequence.  most_keys: no length counts beyond it.
// An item has as many steps as the whole over `target` (or, where that is two, one: twice `target` items then), the last of every row block fewer: at most
// so many items and one for every row block, of which the groups have as many as all sequences' rows and one more each fill, or as many each
// as `largest` sequences do, and the sequences ceil(G / 16) each, a quarter of a workgroup.
extern "C" void velox_shared_prefix_room(int num_seqs, int num_groups, int group, int row_tiles, int target, int largest, long long* items, long long* rows) {
  const long long block_rows = 16LL * row_tiles, own_blocks = (long long)num_seqs * ((group + 15) / 16);
  const long long by_rows = (long long)num_seqs * group / block_rows + num_groups, by_groups = num_groups * (((long long)largest * group + block_rows - 1) / block_rows);
  const long long blocks = by_rows < by_groups ? by_rows : by_groups, most = block_rows > 16 * WAVES ? target : 2LL * target;
  *items = most + blocks + own_blocks / WAVES + 2;
  *rows = most * (block_rows > 16 * WAVES ? block_rows : 16 * WAVES) + blocks * block_rows + own_blocks * 16 + 16 * WAVES;
}
// What a call brings; the host packs it in this order (one argument costs it less than twenty-eight).
struct SharedPrefixCall {
  const void *qkv, *k_cache, *v_cache;
  const int *block_tables, *kv_lens, *group_starts, *shared_lens;
  const float* sinks;
  void* out;
  float *part_o, *part_lse;
  int *directory, *planned;  // planned: 32 int32 for each of `items`, or nullptr with up to 64 sequences and groups
  long long rows_room;
  int items, qkv_stride, table_width, num_seqs, num_groups, nh, nkv, page_shift, pages, most_keys, row_tiles, target, largest, dtype;
  float scale;
  int unused;
};
static_assert(sizeof(SharedPrefixCall) == 14 * 8 + 16 * 4, "as the host packs it");
static_assert(sizeof(Item) == 32 && sizeof(Directory) == 32, "as the host counts their room");

template <typename T>
static int launch(const SharedPrefixCall& c, const Lengths& l, hipStream_t stream) {
  const Cache<T> cache{(const T*)c.k_cache, (const T*)c.v_cache, c.nkv, c.page_shift, (uint32_t)(c.pages - 1)};
  constexpr int MOST = most_row_tiles<T>();
  if (c.row_tiles == 0) {
    shared_prefix_direct_kernel<T><<<dim3(c.nkv, c.num_seqs, (l.group + 15) / 16), THREADS, 0, stream>>>((const T*)c.qkv, c.qkv_stride, cache, c.block_tables, c.table_width, l, c.scale,
                                                                                                  c.sinks, (T*)c.out);
    return (int)hipGetLastError();
  }
  Directory* const directory = (Directory*)c.directory;
  auto kernel = shared_prefix_kernel<T, 1>;
  if constexpr (MOST >= 2) {
    if (c.row_tiles == 2) kernel = shared_prefix_kernel<T, 2>;
  }
  if constexpr (HAS_TALL && sizeof(T) == 2) {
    if (c.row_tiles == TALL) kernel = shared_prefix_kernel<T, TALL>;
  }
  if (l.planned != nullptr) {
    shared_prefix_plan_kernel<<<1, c.num_seqs <= 256 && c.num_groups <= 256 ? 256 : PLAN_THREADS, 0, stream>>>(l, tile_shift<T>(), c.row_tiles == TALL ? step_shift<T, TALL>() : step_shift<T, 1>(), c.items, (Item*)c.planned, directory);
    const int status = (int)hipGetLastError();
    if (status != 0) return status;
  }
  kernel<<<dim3(c.nkv, c.items), THREADS, 0, stream>>>((const T*)c.qkv, c.qkv_stride, cache, c.block_tables, c.table_width, l, c.scale, c.part_o, c.part_lse, directory);
  const int status = (int)hipGetLastError();
  if (status != 0) return status;
  shared_prefix_join_kernel<T><<<dim3((c.nh + JOIN_HEADS - 1) / JOIN_HEADS, l.num_seqs), 64 * JOIN_HEADS, 0, stream>>>(c.nh, l.group, l.rows_room, directory, c.part_o, c.part_lse,
                                                                                                                c.sinks, (T*)c.out);
  return (int)hipGetLastError();
}

extern "C" int velox_shared_prefix_attention(const SharedPrefixCall* call, hipStream_t stream) {
  const SharedPrefixCall& c = *call;
  if (c.num_seqs <= 0) return 0;
  if (c.nkv < 1 || c.nh < 1 || c.nh % c.nkv != 0 || c.page_shift < 3 || c.page_shift > 16 || c.pages < 1 || c.most_keys < 0 || c.most_keys > MOST_KEYS || c.most_keys > (long long)c.table_width << c.page_shift ||
      c.num_groups < 0 || c.num_groups > MOST_GROUPS || c.target < 1 || c.largest < 1 || c.largest > c.num_seqs || c.num_seqs > 65535 || c.items > 65535 || c.rows_room > 0x7fffffffLL) return -1;
  if (!has_row_tiles(c.row_tiles, c.dtype)) return -1;
  const int group = c.nh / c.nkv;
  if (c.row_tiles > 0) {
    long long least_items, least_rows;
    velox_shared_prefix_room(c.num_seqs, c.num_groups, group, c.row_tiles, c.target, c.largest, &least_items, &least_rows);
    if (c.items < least_items || c.rows_room < least_rows) return -1;
    if (c.planned == nullptr && (c.num_seqs > 64 || c.num_groups > 64)) return -1;
  }
  const Lengths l{c.kv_lens, c.group_starts, c.shared_lens, (const Item*)c.planned, c.num_seqs, c.num_groups, group, 16 * c.row_tiles, c.target, c.most_keys, c.largest, (int)c.rows_room};
  return c.dtype == VELOX_BF16 ? launch<bf16_t>(c, l, stream) : launch<float>(c, l, stream);
}
