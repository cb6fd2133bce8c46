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
// once; the second part is each sequence's own, G rows against its keys.
//
// Both parts are cut into items of about equally many keys (see `Plan`), one workgroup each and all in one launch; a second
// kernel joins what the items leave.  A workgroup's four waves take 32 keys in turn, each straight from the cache into the
// operands of matrix instructions, the next tile in flight while one is multiplied: no wave shares a key with another, so
// nothing is staged and no barrier stands in the loop.  Rows are held as tiles of 16, RT of them in every wave.
//
// Matrix cores: S^T[key, row] = K Q^T and O^T[channel, row] = V^T P^T, both with 16 x 16 results.  For a block of KB contraction
// indices (32 in bfloat16, 16 in float32) lane (g = lane / 16, i = lane % 16) holds 16 bytes of row or column i, those of place g; a result is rows
// 4 g .. 4 g + 3 of column i.  In bfloat16 row 4 q + j of the tile's score tile u (q, j < 4) is key 8 q + 4 u + j, so that a lane's
// scores of both are those of keys 8 g .. 8 g + 7: the operand of the second product, and one load of V^T.
#include "common.h"

#ifndef VELOX_HEAD_DIM
#error "build with -DVELOX_HEAD_DIM=<head size>"
#endif
constexpr int D = VELOX_HEAD_DIM;
static_assert(D % 16 == 0 && D >= 16 && D <= 256, "head size must be a multiple of 16 between 16 and 256");

constexpr int TILE = 32;                 // keys a wave takes at a time
constexpr int WAVES = 4;
constexpr int STEP = TILE * WAVES;       // keys a workgroup takes at a time
constexpr int MOST_GROUPS = 1024;

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

template <typename T> struct Block;
template <> struct Block<bf16_t> {
  static constexpr int KB = 32, VEC = 8;
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
// than its group shares, and one that is alone in its group or in none, shares nothing.  The steps of STEP keys of all items
// together over `target` workgroups are what one item may have; a group's rows are cut into blocks of `block_rows`, a
// sequence's G rows into blocks of 16.
struct Lengths {
  const int* kv_lens;
  const int* group_starts;
  const int* shared_lens;
  int num_seqs, num_groups, group, block_rows, target;  // group: query heads of a KV head
  int most;                                             // keys a table has room for
};

struct Groups {  // in LDS
  int start[MOST_GROUPS], end[MOST_GROUPS], shared[MOST_GROUPS];
};

__device__ __forceinline__ int clamped(int v, int lo, int hi) { return v < lo ? lo : (v > hi ? hi : v); }

__device__ __forceinline__ int keys_of(const Lengths& l, int b) { return clamped(l.kv_lens[b], 0, l.most); }

__device__ __forceinline__ void load_groups(const Lengths& l, Groups& groups) {
  for (int g = threadIdx.x; g < l.num_groups; g += blockDim.x) {
    const int start = clamped(l.group_starts[g], 0, l.num_seqs), end = clamped(l.group_starts[g + 1], start, l.num_seqs);
    groups.start[g] = start;
    groups.end[g] = end;
    groups.shared[g] = end - start > 1 ? clamped(l.shared_lens[g], 0, keys_of(l, start)) : 0;
  }
  __syncthreads();
}

struct Own { int group, from, to; };  // a sequence's own keys [from, to); group: whose shared keys it has, or -1
__device__ __forceinline__ Own own_of(const Lengths& l, const Groups& groups, int b) {
  const int len = keys_of(l, b);
  int lo = -1, hi = l.num_groups;  // the last group that begins at b or before
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (groups.start[mid] <= b) lo = mid;
    else hi = mid;
  }
  const bool shares = lo >= 0 && b < groups.end[lo < 0 ? 0 : lo] && groups.shared[lo < 0 ? 0 : lo] > 0 && groups.shared[lo < 0 ? 0 : lo] <= len;
  return Own{shares ? lo : -1, shares ? groups.shared[lo] : 0, len};
}
__device__ __forceinline__ int steps_between(int from, int to) { return to > from ? (to - from / TILE * TILE + STEP - 1) / STEP : 0; }

__device__ __forceinline__ int wave_add(int v) {
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1) v += __shfl_xor(v, offset, VELOX_WAVE);
  return v;
}
__device__ __forceinline__ int wave_add_up_to(int v) {  // v plus those of the lanes before
#pragma unroll
  for (int offset = 1; offset < 64; offset <<= 1) {
    const int w = __shfl_up(v, offset, VELOX_WAVE);
    if ((int)(threadIdx.x & 63) >= offset) v += w;
  }
  return v;
}

__device__ __forceinline__ int blocks_of(const Lengths& l, const Groups& groups, int g) {
  return groups.shared[g] > 0 ? ((groups.end[g] - groups.start[g]) * l.group + l.block_rows - 1) / l.block_rows : 0;
}

// steps of one item (the whole wave takes part)
__device__ __forceinline__ int steps_per_item(const Lengths& l, const Groups& groups) {
  const int lane = threadIdx.x & 63, own_blocks = (l.group + 15) / 16;
  int total = 0;
  for (int g = lane; g < l.num_groups; g += 64) total += blocks_of(l, groups, g) * steps_between(0, groups.shared[g]);
  for (int b = lane; b < l.num_seqs; b += 64) {
    const Own own = own_of(l, groups, b);
    total += own_blocks * steps_between(own.from, own.to);
  }
  total = wave_add(total);
  return max(1, (total + l.target - 1) / l.target);
}

// Items in their order: group by group, of each the parts of the keys, of each part the row blocks; then sequence by sequence the
// same.  `before` of either: the items before it.
struct Item { int group, sequence, block, part, per; };  // group >= 0: of a group's shared keys; else sequence >= 0; else none

__device__ __forceinline__ Item find_item(const Lengths& l, const Groups& groups, int item) {
  const int lane = threadIdx.x & 63, own_blocks = (l.group + 15) / 16;
  const int per = steps_per_item(l, groups);
  int before = 0;
  for (int base = 0; base < l.num_groups; base += 64) {
    const int g = base + lane;
    const int blocks = g < l.num_groups ? blocks_of(l, groups, g) : 0;
    const int items = blocks > 0 ? blocks * ((steps_between(0, groups.shared[g]) + per - 1) / per) : 0;
    const int upto = wave_add_up_to(items);
    const uint64_t holds = __ballot(before + upto > item);
    if (holds != 0) {
      const int at = __ffsll((unsigned long long)holds) - 1;
      const int place = item - (before + __builtin_amdgcn_readlane(upto - items, at)), row_blocks = __builtin_amdgcn_readlane(blocks, at);
      return Item{base + at, -1, place % row_blocks, place / row_blocks, per};
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  for (int base = 0; base < l.num_seqs; base += 64) {
    const int b = base + lane;
    int items = 0;
    if (b < l.num_seqs) {
      const Own own = own_of(l, groups, b);
      items = own_blocks * ((steps_between(own.from, own.to) + per - 1) / per);
    }
    const int upto = wave_add_up_to(items);
    const uint64_t holds = __ballot(before + upto > item);
    if (holds != 0) {
      const int at = __ffsll((unsigned long long)holds) - 1;
      const int place = item - (before + __builtin_amdgcn_readlane(upto - items, at));
      return Item{-1, base + at, place % own_blocks, place / own_blocks, per};
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return Item{-1, -1, 0, 0, per};
}

// ---- one item ---------------------------------------------------------------------------------------------------------------
template <typename T> struct Cache {
  const T* k;
  const T* v;
  int nkv, page_shift;
  uint32_t last_page;  // (an id beyond it, which no table should hold, reads this one)
};

// Row tiles of queries against the keys [lo, hi) of a table's sequence; what they leave goes to part_o[row][D] and part_lse[row].
// query(row) is the address of a row's query, or nullptr; rows are [first_row, first_row + 16 RT).
template <typename T, int RT, int DEPTH, typename QueryOf>
__device__ __forceinline__ void work_item(const Cache<T>& cache, int kvh, const int* __restrict__ table, int lo, int hi, float scale, QueryOf query,
                                          float* __restrict__ part_o, float* __restrict__ part_lse, char* smem) {
  typedef Block<T> B;
  constexpr int KB = B::KB, VEC = B::VEC;
  constexpr int NQB = (D + KB - 1) / KB;   // contraction blocks of K Q^T (beyond the head size: zeros)
  constexpr int NKB = TILE / KB;           // of V^T P^T
  constexpr int NC = D / 16;
  constexpr int IDS = NKB;                 // page ids a lane needs for a tile's keys, and as many for its values
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, i = lane & 15;
  const int page_size = 1 << cache.page_shift;

  const int tile_lo = lo / TILE, tile_hi = (hi + TILE - 1) / TILE;
  const int mine = tile_lo + wave;

  // Keys beyond either end are read from the nearest place inside: their scores are masked and their values zeroed.
  auto key_at = [&](int tile, int u) { return clamped(TILE * tile + B::key_row(u, i), lo, hi - 1); };
  auto value_at = [&](int tile, int kb) { return clamped(TILE * tile + KB * kb + VEC * g, lo & ~(VEC - 1), (hi - 1) & ~(VEC - 1)); };
  struct Ids { uint32_t k[IDS], v[IDS]; };
  auto load_ids = [&](Ids& ids, int tile) {
#pragma unroll
    for (int a = 0; a < IDS; ++a) {
      ids.k[a] = min((uint32_t)table[key_at(tile, a) >> cache.page_shift], cache.last_page);  // (bfloat16: a lane's keys of both score tiles lie in one run of eight)
      ids.v[a] = min((uint32_t)table[value_at(tile, a) >> cache.page_shift], cache.last_page);
    }
  };
  struct Tile { float4_t k[2][NQB], v[NC][NKB]; };
  auto load_tile = [&](Tile& x, const Ids& ids, int tile) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int n = key_at(tile, u);
      const T* p = cache.k + ((((size_t)ids.k[IDS == 1 ? 0 : u] * cache.nkv + kvh) << cache.page_shift) + (n & (page_size - 1))) * D + VEC * g;
#pragma unroll
      for (int cb = 0; cb < NQB; ++cb) {
        // (of a block that reaches beyond the head size, lanes there read the row's beginning and hold zeros)
        const bool inside = D % KB == 0 || KB * cb + VEC * g < D;
        x.k[u][cb] = *reinterpret_cast<const float4_t*>(p + (inside ? KB * cb : -VEC * g));
        if (!inside) x.k[u][cb] = float4_t{0.f, 0.f, 0.f, 0.f};
      }
    }
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb) {
      const int n = value_at(tile, kb);
      const T* p = cache.v + ((((size_t)ids.v[kb] * cache.nkv + kvh) * D + i) << cache.page_shift) + (n & (page_size - 1));
#pragma unroll
      for (int c = 0; c < NC; ++c) x.v[c][kb] = *reinterpret_cast<const float4_t*>(p + ((size_t)(16 * c) << cache.page_shift));
    }
  };

  float4_t qf[RT][NQB], acc[RT][NC];
  float m_i[RT], l_i[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const T* q = query(16 * rt + i);
#pragma unroll
    for (int cb = 0; cb < NQB; ++cb) {
      qf[rt][cb] = float4_t{0.f, 0.f, 0.f, 0.f};
      if (q != nullptr && (D % KB == 0 || KB * cb + VEC * g < D)) qf[rt][cb] = *reinterpret_cast<const float4_t*>(q + KB * cb + VEC * g);
    }
    m_i[rt] = -INFINITY;
    l_i[rt] = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[rt][c] = float4_t{0.f, 0.f, 0.f, 0.f};
  }
  const float scale_eff = scale * B::SCALE;

  auto compute = [&](Tile& x, int tile) {
    const int n0 = TILE * tile;
    const bool whole = n0 >= lo && n0 + TILE <= hi;  // (the same for the whole wave)
    if (!whole) {
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) {
        const int n = n0 + KB * kb + VEC * g;
#pragma unroll
        for (int c = 0; c < NC; ++c) B::mask(x.v[c][kb], lo - n, hi - n);
      }
    }
    float4_t pf[RT][NKB];
    float alpha[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float4_t s[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        s[u] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int cb = 0; cb < NQB; ++cb) s[u] = B::mma(x.k[u][cb], qf[rt][cb], s[u]);
      }
      if (!whole) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int n = n0 + B::first_score(u, g) + j;
            s[u][j] = n >= lo && n < hi ? s[u][j] : -INFINITY;
          }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = fmaxf(mx, s[u][j]);
      mx = fmaxf(mx, __shfl_xor(mx, 16, VELOX_WAVE));
      mx = fmaxf(mx, __shfl_xor(mx, 32, VELOX_WAVE));
      const float m_new = fmaxf(m_i[rt], mx * scale_eff);  // (the scale is positive)
      const float m_safe = m_new == -INFINITY ? 0.f : m_new;
      alpha[rt] = m_i[rt] == -INFINITY ? 0.f : B::exp_of(m_i[rt] - m_safe);
      float sum = 0.f;
      float p[2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          p[u][j] = B::exp_of(fmaf(s[u][j], scale_eff, -m_safe));
          sum += p[u][j];
        }
      if constexpr (sizeof(T) == 2) {
        bf16x8_t e;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j) e[4 * u + j] = (bf16_t)p[u][j];  // probabilities are rounded to the values' type for the product
        pf[rt][0] = __builtin_bit_cast(float4_t, e);
      } else {
#pragma unroll
        for (int u = 0; u < 2; ++u) pf[rt][u < NKB ? u : 0] = float4_t{p[u][0], p[u][1], p[u][2], p[u][3]};
      }
      l_i[rt] = l_i[rt] * alpha[rt] + sum;  // of this lane's keys; the four lane groups are added up at the end
      m_i[rt] = m_new;
    }
    // the output is rescaled only where a row's maximum moved, which is the exception after a row's first keys
    bool moved = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) moved = moved || alpha[rt] != 1.f;
    if (__ballot(moved) != 0ull) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int c = 0; c < NC; ++c) acc[rt][c] = acc[rt][c] * alpha[rt];
    }
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) acc[rt][c] = B::mma(x.v[c][kb], pf[rt][kb], acc[rt][c]);
  };

  if (mine < tile_hi) {
    const int last = mine + (tile_hi - 1 - mine) / WAVES * WAVES;  // this wave's last tile
    Ids ids;
    load_ids(ids, mine);
    if constexpr (DEPTH == 2) {
      // page ids two tiles ahead, keys and values one; what is asked for beyond the last tile is the last tile again
      Tile ring[2];
      load_tile(ring[0], ids, mine);
      load_ids(ids, min(mine + WAVES, last));
      auto step = [&](int tile, Tile& now, Tile& next) {
        const int ahead = min(tile + WAVES, last), further = min(tile + 2 * WAVES, last);
        Ids later;
        load_ids(later, further);
        load_tile(next, ids, ahead);
        ids = later;
        compute(now, tile);
      };
      for (int tile = mine; tile < tile_hi; tile += 2 * WAVES) {
        step(tile, ring[0], ring[1]);
        if (tile + WAVES < tile_hi) step(tile + WAVES, ring[1], ring[0]);
      }
    } else {
      Tile x;
      for (int tile = mine; tile < tile_hi; tile += WAVES) {
        load_tile(x, ids, tile);
        load_ids(ids, min(tile + WAVES, last));
        compute(x, tile);
      }
    }
  }

  // ---- the four waves' results, a row tile at a time ----
  float4_t* const acc_all = reinterpret_cast<float4_t*>(smem);                        // [wave][channel tile][lane]
  float* const m_all = reinterpret_cast<float*>(smem + WAVES * NC * 64 * 16);         // [wave][16 RT]
  float* const l_all = m_all + WAVES * 16 * RT;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    l_i[rt] += __shfl_xor(l_i[rt], 16, VELOX_WAVE);
    l_i[rt] += __shfl_xor(l_i[rt], 32, VELOX_WAVE);
    if (g == 0) {
      m_all[wave * 16 * RT + 16 * rt + i] = m_i[rt];
      l_all[wave * 16 * RT + 16 * rt + i] = l_i[rt];
    }
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    if (rt > 0) __syncthreads();
#pragma unroll
    for (int c = 0; c < NC; ++c) acc_all[(wave * NC + c) * 64 + lane] = acc[rt][c];
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
    const float inv = total > 0.f ? 1.f / total : 1.f;
    for (int c = wave; c < NC; c += WAVES) {
      float4_t sum = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < WAVES; ++w) sum += acc_all[(w * NC + c) * 64 + lane] * weight[w];
      *reinterpret_cast<float4_t*>(part_o + (size_t)(16 * rt + i) * D + 16 * c + 4 * g) = sum * inv;
    }
    if (wave == 0 && g == 0) part_lse[16 * rt + i] = total > 0.f ? top * B::LN_UNIT + logf(total) : -INFINITY;
  }
}

template <int RT> constexpr int epilogue_bytes() { return WAVES * (D / 16) * 64 * 16 + 2 * WAVES * 16 * RT * 4; }

// part_o: [item][KV head][block_rows][D], part_lse: [item][KV head][block_rows]
template <typename T, int RT, int DEPTH>
__global__ void __launch_bounds__(64 * WAVES, 1) shared_prefix_kernel(const T* __restrict__ qkv, int qkv_stride, const Cache<T> cache, const int* __restrict__ block_tables,
                                                                      int table_width, const Lengths l, float scale, float* __restrict__ part_o,
                                                                      float* __restrict__ part_lse) {
  __shared__ __attribute__((aligned(16))) char smem[sizeof(Groups) > epilogue_bytes<RT>() ? sizeof(Groups) : epilogue_bytes<RT>()];
  Groups& groups = *reinterpret_cast<Groups*>(smem);
  load_groups(l, groups);
  const int kvh = blockIdx.x;
  const Item item = find_item(l, groups, blockIdx.y);
  if (item.group < 0 && item.sequence < 0) return;  // (uniform over the workgroup)
  const size_t slot = ((size_t)blockIdx.y * cache.nkv + kvh) * (16 * RT);
  float* const o = part_o + slot * D;
  float* const lse = part_lse + slot;
  const int group_heads = l.group;
  if (item.group >= 0) {
    const int start = groups.start[item.group], rows = (groups.end[item.group] - start) * group_heads, shared = groups.shared[item.group];
    __syncthreads();  // (the groups' place is used again)
    const int first_row = item.block * 16 * RT;
    const int lo = item.part * item.per * STEP, hi = min(lo + item.per * STEP, shared);
    auto query = [&](int r) -> const T* {
      const int row = first_row + r;
      return row < rows ? qkv + (size_t)(start + row / group_heads) * qkv_stride + (size_t)(kvh * group_heads + row % group_heads) * D : nullptr;
    };
    work_item<T, RT, DEPTH>(cache, kvh, block_tables + (size_t)start * table_width, lo, hi, scale, query, o, lse, smem);
  } else {
    const Own own = own_of(l, groups, item.sequence);
    __syncthreads();
    const int base = own.from / TILE * TILE + item.part * item.per * STEP;
    const int lo = max(base, own.from), hi = min(base + item.per * STEP, own.to);
    auto query = [&](int r) -> const T* {
      const int row = item.block * 16 + r;
      return row < group_heads ? qkv + (size_t)item.sequence * qkv_stride + (size_t)(kvh * group_heads + row) * D : nullptr;
    };
    work_item<T, 1, 2 * sizeof(T) * D <= 1024 ? 2 : 1>(cache, kvh, block_tables + (size_t)item.sequence * table_width, lo, hi, scale, query, o, lse, smem);
  }
}

// A workgroup per (sequence, KV head): the items that hold its rows, joined.  A sink adds exp(sink) to the denominator.
constexpr int MERGE_THREADS = 256;
template <typename T>
__global__ void __launch_bounds__(MERGE_THREADS) shared_prefix_merge_kernel(const Lengths l, int nkv, const float* __restrict__ part_o, const float* __restrict__ part_lse,
                                                                            const float* __restrict__ sinks, T* __restrict__ out, int items_room) {
  __shared__ Groups groups;
  load_groups(l, groups);
  const int kvh = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 63, own_blocks = (l.group + 15) / 16;
  const int per = steps_per_item(l, groups);
  const Own own = own_of(l, groups, b);
  // items before this sequence's group, of all groups, and of the sequences before this one
  int before_group = 0, before_own = 0;
  for (int g = lane; g < l.num_groups; g += 64) {
    const int items = blocks_of(l, groups, g) * ((steps_between(0, groups.shared[g]) + per - 1) / per);
    before_own += items;
    before_group += g < own.group ? items : 0;
  }
  for (int s = lane; s < b; s += 64) {
    const Own other = own_of(l, groups, s);
    before_own += own_blocks * ((steps_between(other.from, other.to) + per - 1) / per);
  }
  before_group = wave_add(before_group);
  before_own = wave_add(before_own);
  const int shared_blocks = own.group >= 0 ? blocks_of(l, groups, own.group) : 0;
  const int shared_parts = own.group >= 0 ? (steps_between(0, own.from) + per - 1) / per : 0;
  const int own_parts = (steps_between(own.from, own.to) + per - 1) / per;
  const int first_row = own.group >= 0 ? (b - groups.start[own.group]) * l.group : 0;
  constexpr int QUADS = D / 4;
  for (int at = threadIdx.x; at < l.group * QUADS; at += MERGE_THREADS) {
    const int h = at / QUADS, channel = at % QUADS * 4;
    const int row = first_row + h;
    auto place_of = [&](int part) -> size_t {  // of this head's row in the part's item
      const int item = part < shared_parts ? before_group + part * shared_blocks + row / l.block_rows : before_own + (part - shared_parts) * own_blocks + h / 16;
      const int r = part < shared_parts ? row % l.block_rows : h % 16;
      return ((size_t)min(item, items_room - 1) * nkv + kvh) * l.block_rows + r;
    };
    float top = -INFINITY, denom = 0.f;
    float4_t acc = float4_t{0.f, 0.f, 0.f, 0.f};
    constexpr int ROUND = 8;
    const int parts = shared_parts + own_parts;
    for (int p0 = 0; p0 < parts; p0 += ROUND) {
      float logs[ROUND];
      float4_t o[ROUND];
#pragma unroll
      for (int j = 0; j < ROUND; ++j) {
        const size_t place = place_of(min(p0 + j, parts - 1));
        logs[j] = p0 + j < parts ? part_lse[place] : -INFINITY;
        o[j] = *reinterpret_cast<const float4_t*>(part_o + place * D + channel);
      }
      float now = top;
#pragma unroll
      for (int j = 0; j < ROUND; ++j) now = fmaxf(now, logs[j]);
      const float safe = now == -INFINITY ? 0.f : now, old = top == -INFINITY ? 0.f : expf(top - safe);
      denom *= old;
      acc = acc * old;
      top = now;
#pragma unroll
      for (int j = 0; j < ROUND; ++j) {
        if (logs[j] == -INFINITY) continue;  // (what was asked for again may be anything)
        const float weight = expf(logs[j] - safe);
        denom += weight;
        acc += o[j] * weight;
      }
    }
    const int head = kvh * l.group + h;
    if (sinks != nullptr && top != -INFINITY) denom += expf(sinks[head] - top);
    const float4_t result = acc * (denom > 0.f ? 1.f / denom : 1.f);
    T* dst = out + ((size_t)b * l.group * nkv + head) * D + channel;
#pragma unroll
    for (int j = 0; j < 4; ++j) dst[j] = from_f32<T>(result[j]);
  }
}

// Row tiles a wave can hold: its registers hold the queries, the output and two tiles of keys and values.
template <typename T> constexpr int most_row_tiles() { return sizeof(T) * D <= 256 ? 4 : sizeof(T) * D <= 512 ? 2 : 1; }

extern "C" int velox_shared_prefix_head_dim() { return D; }
extern "C" int velox_shared_prefix_most_row_tiles(int dtype) { return dtype == VELOX_BF16 ? most_row_tiles<bf16_t>() : most_row_tiles<float>(); }

template <typename T>
static int launch(const void* qkv, int qkv_stride, const void* k_cache, const void* v_cache, const int* block_tables, int table_width, const Lengths& l, int row_tiles,
                  int items, const float* sinks, void* out, float* part_o, float* part_lse, int nkv, int page_shift, int pages, float scale, hipStream_t stream) {
  const Cache<T> cache{(const T*)k_cache, (const T*)v_cache, nkv, page_shift, (uint32_t)(pages - 1)};
  constexpr int DEPTH = sizeof(T) * D <= 512 ? 2 : 1, MOST = most_row_tiles<T>();
  const dim3 grid(nkv, items);
  if (row_tiles == 1) shared_prefix_kernel<T, 1, DEPTH><<<grid, 64 * WAVES, 0, stream>>>((const T*)qkv, qkv_stride, cache, block_tables, table_width, l, scale, part_o, part_lse);
  if constexpr (MOST >= 2) {
    if (row_tiles == 2) shared_prefix_kernel<T, 2, DEPTH><<<grid, 64 * WAVES, 0, stream>>>((const T*)qkv, qkv_stride, cache, block_tables, table_width, l, scale, part_o, part_lse);
  }
  if constexpr (MOST >= 4) {
    if (row_tiles == 4) shared_prefix_kernel<T, 4, DEPTH><<<grid, 64 * WAVES, 0, stream>>>((const T*)qkv, qkv_stride, cache, block_tables, table_width, l, scale, part_o, part_lse);
  }
  const int status = (int)hipGetLastError();
  if (status != 0) return status;
  shared_prefix_merge_kernel<T><<<dim3(nkv, l.num_seqs), MERGE_THREADS, 0, stream>>>(l, nkv, part_o, part_lse, sinks, (T*)out, items);
  return (int)hipGetLastError();
}

// items: at least the most there can be, one more for every row block than its share of `target`: at most num_seqs G / (16 row_tiles) +
// num_groups of the groups' and num_seqs ceil(G / 16) of the sequences'.  most_keys: no length counts beyond it.  part_o: float32 [items, nkv, 16 row_tiles, D], part_lse the same without D.
extern "C" int velox_shared_prefix_attention(const void* qkv, int qkv_stride, const void* k_cache, const void* v_cache, const int* block_tables, int table_width,
                                             const int* kv_lens, const int* group_starts, const int* shared_lens, int num_seqs, int num_groups, int nh, int nkv,
                                             int page_shift, int pages, int most_keys, float scale, int row_tiles, int target, int items, const float* sinks, void* out, float* part_o, float* part_lse,
                                             int dtype, hipStream_t stream) {
  if (num_seqs <= 0) return 0;
  if (nkv < 1 || nh % nkv != 0 || page_shift < 3 || pages < 1 || most_keys < 0 || most_keys > (long long)table_width << page_shift || num_groups < 0 || num_groups > MOST_GROUPS || target < 1 || num_seqs > 65535 || items > 65535) return -1;
  if (row_tiles < 1 || row_tiles == 3 || row_tiles > velox_shared_prefix_most_row_tiles(dtype)) return -1;
  const int group = nh / nkv;
  const long long most = (long long)target + (long long)num_seqs * group / (16 * row_tiles) + num_groups + (long long)num_seqs * ((group + 15) / 16);
  if (items < most) return -1;
  const Lengths l{kv_lens, group_starts, shared_lens, num_seqs, num_groups, group, 16 * row_tiles, target, most_keys};
  if (dtype == VELOX_BF16)
    return launch<bf16_t>(qkv, qkv_stride, k_cache, v_cache, block_tables, table_width, l, row_tiles, items, sinks, out, part_o, part_lse, nkv, page_shift, pages, scale, stream);
  return launch<float>(qkv, qkv_stride, k_cache, v_cache, block_tables, table_width, l, row_tiles, items, sinks, out, part_o, part_lse, nkv, page_shift, pages, scale, stream);
}
