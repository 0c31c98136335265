// Attention of a batch whose sequences begin with the same keys: the shared keys are read once for all rows, then each sequence's own.
//
//   s = scale q . k (capped: c tanh(s / c)),  w = exp(s - m),  o = sum w v / sum w     over the keys up to the query's position.
// A softmax over disjoint ranges of keys joins: with each range's maximum m_i, l_i = sum exp(s - m_i) and o_i = sum exp(s - m_i) v,
// m = max m_i, l = sum l_i exp(m_i - m), o = sum o_i exp(m_i - m) / l.  So the work is cut into items, each some rows by some keys of one
// key/value head, that leave (m, l, o) in the workspace in float32; a second launch joins a row's parts in a fixed order.
// A row is a token and a head of the group: rows of one key/value head are numbered token by token, so that the rows of all sequences
// multiply the shared keys in one product, and a sequence's own keys are met by its own rows alone.
//
// An item is a block of four waves, two blocks a CU: up to 128 rows in tiles of 32, a wave a tile; with fewer rows the waves share out the keys of
// a stage and join at the end.  Keys and values travel straight into LDS, a stage ahead, one barrier a stage:
//   S^T[key, row] = K . Q^T,   O^T[dim, row] += V^T . P^T       32x32 matrix instructions, queries, sums and statistics in registers.
// The product S^T leaves a lane 16 keys of one row.  bfloat16: key rows lie in LDS with bits 2 and 3 of their number swapped, which
// makes a lane's keys two runs of eight: what the second product takes as its operand.  float32: runs of four, as the float32
// instruction takes them; nothing is rounded before the result.  Values lie in LDS as the second product reads them, runs of two pieces
// of 16 bytes a dimension: 1 KB a read and 1 KB a load, whose lanes' addresses are one number a lane beside scalars.
// Weights are rounded to bfloat16 for the product with the values (half a step each); the sum of the weights is of the unrounded ones.
//
// Heads of 128, bfloat16: 16 sequences of one query behind 32,000 keys (40 heads in 8 groups) 45.0 us, 3.3 TB/s; 64 of 1 to 5 queries behind
// 8,192 keys and 64 to 1,024 own (28 heads in 4 groups) 55 us, 430 TFLOP/s.  Neither bytes nor products bound these: of the second's 46.6 us in
// the first launch the matrix cores work 10 and the vector unit 11, and waves wait two fifths of their time.  A stage of 64 keys by 128 rows
// takes 1.35 us for a block alone on the chip, 2.2 with one on every CU and 3.0 each with two, which is 1.36 times the work of one; but 352 blocks
// of 16 stages leave 160 of the 256 CUs with one.  Small batches are bound by two launches and the trips from table to page to
// product: four sequences behind 500 keys 9.4 + 3.9 us.
#include <type_traits>

#include "mfma.h"
#include "sprout_hip.h"

namespace sprout {

namespace {

constexpr float kLog2E = 1.4426950408889634f;
constexpr float kNothingYet = -1.0e30f;      // running maximum before any key: finite, so that no inf - inf arises
constexpr float kMaxMoves = 8.0f;            // the running maximum follows the true one when that lies further above it (log2): until
                                             // then weights reach 2^8 at most, which float32 and bfloat16 hold as well as 1
constexpr int kSharedTile = 16;              // queries of one entry of the tile list

struct SharedArgs {
  const void *q, *k_pool, *v_pool;
  const int32_t *block_tables, *prefix_table, *q_start, *q_len, *ctx_len, *tiles;
  float *part_o, *part_ml;
  const float* sinks;
  int q_stride, max_blocks, prefix, tokens, n_tiles, nq, nkv, hd, page_size, num_pages;
  int page_shift;                                              // page_size == 1 << page_shift (16-byte pieces only)
  int prefix_splits, prefix_keys, row_blocks, block_rows;      // shared keys: parts, keys of each, blocks of rows, rows of each
  int own_splits, own_keys, own_rows;                          // own keys: parts, keys of each, blocks of 128 rows of an entry
  float scale2, cap;                                           // scale in log2 units; with a cap (0: none) twice that over the cap
};

// cap tanh(x) in log2 units, of 2 x in log2 units: tanh x = 1 - 2 / (exp(2 x) + 1), off by some 2^-23; below 0.3, where that is more than
// a few units of the result's last place and the cap may be far above the scores, the Taylor polynomial (5e-8 of the value).
__device__ __forceinline__ float capped(float x2, float cap) {
  const float x = x2 * 0.34657359f, y = x * x;
  const float near = x * fmaf(y, fmaf(y, fmaf(y, fmaf(y, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f);
  const float far = 1.f - 2.f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x2) + 1.f);
  return cap * kLog2E * (fabsf(x) < 0.3f ? near : far);
}

template <typename E> struct Numbers;
template <> struct Numbers<bf16_t> { static constexpr int kChunk = 8; };
template <> struct Numbers<float> { static constexpr int kChunk = 4; };

// Where piece c (16 bytes) of a row of C pieces lies: 16-byte reads of a half-wave are served in groups of lanes {0-3, 12-15, 20-27} and
// the others, 256 bytes each; the 16 rows of a group meet 16 different places of these.
template <int C> __device__ __forceinline__ int place_in_row(int row, int c) {
  return C % 16 == 0 ? c ^ (row & 15) : C % 8 == 0 ? c ^ ((row ^ (row >> 3)) & 7) : c ^ ((row >> 2) & 3);
}
__device__ __forceinline__ int swap23(int key) { return (key & ~12) | ((key & 4) << 1) | ((key & 8) >> 1); }
__device__ __forceinline__ float larger(float a, float b) { return __builtin_amdgcn_fmed3f(a, b, INFINITY); }
// The largest of three in one instruction (v_maximum3_f32; NaN if one of them is).
__device__ __forceinline__ float largest(float a, float b, float c) { return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c); }
__device__ __forceinline__ float other_half(float x) {      // lane ^ 32's
  const unsigned u = __float_as_uint(x);
  const auto f = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float((threadIdx.x & 32) ? f[0] : f[1]);
}

// Where number j of a piece lies in its words, and whether it is NaN or infinite.
template <typename E> __device__ __forceinline__ uint32_t bits_of(int j) { return std::is_same<E, float>::value ? ~0u : (j & 1) ? 0xffff0000u : 0x0000ffffu; }
template <typename E> __device__ __forceinline__ bool not_finite(uint32_t word, int j) {
  const uint32_t exponent = (std::is_same<E, float>::value ? 0x7f800000u : 0x7f807f80u) & bits_of<E>(j);
  return (word & exponent) == exponent;
}

// c += a . b of one piece a lane: bfloat16 one instruction of 16, float32 four of 2.
__device__ __forceinline__ floatx16 piece_product(uint4 a, uint4 b, floatx16 c, bf16_t) { return mfma32(as_bf16x8(a), as_bf16x8(b), c); }
__device__ __forceinline__ floatx16 piece_product(uint4 a, uint4 b, floatx16 c, float) {
  c = mfma32_f32(__uint_as_float(a.x), __uint_as_float(b.x), c);
  c = mfma32_f32(__uint_as_float(a.y), __uint_as_float(b.y), c);
  c = mfma32_f32(__uint_as_float(a.z), __uint_as_float(b.z), c);
  return mfma32_f32(__uint_as_float(a.w), __uint_as_float(b.w), c);
}
// Weights 4 or 8 times `part` on of a lane's sixteen, as an operand.
__device__ __forceinline__ uint4 weights_of(const floatx16& s, int part, bf16_t) {
  return make_uint4(pack_bf16x2(s[8 * part], s[8 * part + 1]), pack_bf16x2(s[8 * part + 2], s[8 * part + 3]),
                    pack_bf16x2(s[8 * part + 4], s[8 * part + 5]), pack_bf16x2(s[8 * part + 6], s[8 * part + 7]));
}
__device__ __forceinline__ uint4 weights_of(const floatx16& s, int part, float) {
  return make_uint4(__float_as_uint(s[4 * part]), __float_as_uint(s[4 * part + 1]), __float_as_uint(s[4 * part + 2]), __float_as_uint(s[4 * part + 3]));
}

constexpr int kWaves = 4, kThreads = 64 * kWaves;
// Keys of a stage, of which two lie in LDS: 32 KB (heads of 256 in float32: 64), at most 128 keys.
template <typename E, int HD> constexpr int stage_keys() { return HD * int(sizeof(E)) <= 128 ? 128 : HD * int(sizeof(E)) <= 256 ? 64 : 32; }

// E: the numbers' type, HD: dimensions held (the head's size or the next one up, zeros behind it).  RUNS: pages are a power of two of 16 tokens
// at least and rows are whole pieces of 16 bytes, so that a wave's loads are runs of one page each; otherwise numbers are loaded one by one.
template <typename E, int HD, bool RUNS>
__global__ __launch_bounds__(kThreads, HD * sizeof(E) <= 256 ? 2 : 1) void attention_shared_kernel(SharedArgs a) {
  constexpr int EPC = Numbers<E>::kChunk, KEYS = stage_keys<E, HD>(), KC = HD / EPC, TILES = KEYS / 32, DT = HD / 32, STEPS = HD / (2 * EPC);
  constexpr int PSTEPS = 32 / (2 * EPC), GROUP = 2 * EPC, HALF = KEYS * HD * int(sizeof(E)), STAGE = 2 * HALF, LOADS = HALF / (1024 * kWaves);
  constexpr bool kF32 = std::is_same<E, float>::value;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];

  // ---- which item: rows first_row .. + rows of key/value head g, keys lo .. hi - 1, part `slot`
  const int G = a.nq / a.nkv;
  const int prefix_items = (a.prefix_splits * a.nkv + 7) / 8 * 8 * a.row_blocks;
  int g, first_row, rows, lo, hi, slot, seq = -1, first_pos = 0, first_token = 0;
  const int32_t* table;
  if (int(blockIdx.x) < prefix_items) {
    // blocks go round the 8 XCDs: those that read the same keys are 8 apart, so that the keys come to one L2
    const int local = blockIdx.x / 8, rb = local % a.row_blocks, unit = local / a.row_blocks * 8 + blockIdx.x % 8;
    if (unit >= a.prefix_splits * a.nkv) return;
    g = unit % a.nkv;
    slot = unit / a.nkv;
    first_row = rb * a.block_rows;
    rows = min(a.block_rows, a.tokens * G - first_row);
    lo = slot * a.prefix_keys;
    hi = min(a.prefix, lo + a.prefix_keys);
    table = a.prefix_table;
  } else {
    int i = blockIdx.x - prefix_items;
    const int rb = i % a.own_rows;
    i /= a.own_rows;
    g = i % a.nkv;
    i /= a.nkv;
    const int entry = i % a.n_tiles, part = i / a.n_tiles;
    const auto scalar = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    seq = scalar(a.tiles[2 * entry]);
    const int q_off = scalar(a.tiles[2 * entry + 1]), len = scalar(a.q_len[seq]), ctx = scalar(a.ctx_len[seq]);
    const int queries = min(kSharedTile, len - q_off);
    first_token = scalar(a.q_start[seq]) + q_off;
    first_row = first_token * G + 128 * rb;
    rows = min(128, queries * G - 128 * rb);
    if (rows <= 0) return;
    first_pos = ctx - len + q_off;
    slot = a.prefix_splits + part;
    lo = a.prefix + part * a.own_keys;
    hi = min(min(first_pos + queries, lo + a.own_keys), a.max_blocks * a.page_size);
    table = a.block_tables + size_t(seq) * a.max_blocks;
  }
  const bool own = seq >= 0;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, li = lane & 31, lk = lane >> 5;
  const int row_tiles = (rows + 31) / 32;
  const int shift = row_tiles == 1 ? 0 : row_tiles == 2 ? 1 : 2;      // 1, 2 or 4 waves side by side along the rows
  const int tile = wave & ((1 << shift) - 1), share = wave >> shift, shares = kWaves >> shift;
  const bool live = tile < row_tiles;
  const int row = first_row + min(32 * tile + li, rows - 1), token = row / G, head = g * G + (row - token * G);
  const size_t place = size_t(token) * a.nq + head;
  const bool real = 32 * tile + li < rows;
  float* ml = a.part_ml + (size_t(slot) * a.tokens * a.nq + place) * 2;
  if (hi <= lo) {      // own keys that end before this part: said to the joining launch, which reads every part's statistics
    if (live && share == 0 && real && lk == 0) { ml[0] = kNothingYet; ml[1] = 0.f; }
    return;
  }

  const int last = own ? min(first_pos + token - first_token, hi - 1) : hi - 1;      // the last key that the row sees
  const int seen_by_all = own ? min(first_pos + 1, hi) : hi;                          // keys before this one are seen by every row

  // ---- a stage's way into LDS: key rows, 16-byte pieces placed as `place_in_row` says, then values [GROUP keys][dimension][2 pieces]
  const int first_key = lo / 16 * 16;
  const bool whole = a.hd == HD;
  auto page_of = [&](int index) __attribute__((always_inline)) {
    return size_t(min(max(table[index], 0), a.num_pages - 1)) * a.nkv + g;      // a bad table entry must not become a wild address
  };
  // RUNS: what a lane adds to the run's start, and whether there is anything of the head in its piece
  uint32_t k_lane[RUNS ? LOADS : 1], v_lane = 0;
  bool k_there[RUNS ? LOADS : 1], v_there[RUNS ? LOADS : 1];
  if (RUNS) {
    v_lane = uint32_t((lane >> 1) * a.page_size + (lane & 1) * EPC) * sizeof(E);
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int i = 64 * (wave + kWaves * u) + lane, r = i / KC, c = place_in_row<KC>(r, i % KC);
      k_lane[u] = uint32_t(((kF32 ? r : swap23(r)) & 15) * a.hd + c * EPC) * sizeof(E);
      k_there[u] = c * EPC < a.hd;
      v_there[u] = 32 * ((wave + kWaves * u) % DT) + (lane >> 1) < a.hd;
    }
    if (!whole) {      // what lies behind the head stays zero
      for (int i = threadIdx.x; i < 2 * STAGE / 16; i += kThreads) *reinterpret_cast<uint4*>(lds + 16 * i) = make_uint4(0, 0, 0, 0);
      __syncthreads();
    }
  }
  const uint32_t lds_base = uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char*)lds));
  // Page numbers come a stage before they are used: their trips would otherwise stand before every stage's loads.  Lane u holds where load u of
  // the wave's keys starts, lane 16 + u the same of its values: a lane's arithmetic serves all loads, a load takes its start with two moves.
  const unsigned char* pools = static_cast<const unsigned char*>(lane < 16 ? a.k_pool : a.v_pool) + size_t(g) * a.page_size * a.hd * sizeof(E);
  const uint64_t page_bytes = uint64_t(a.nkv) * a.page_size * a.hd * sizeof(E);
  const int my_load = wave + kWaves * min(lane & 15, LOADS - 1);
  const int my_key = lane < 16 ? 64 * my_load / KC / 16 * 16 : my_load / DT * GROUP, my_dim = (32 * (my_load % DT)) << a.page_shift;
  int32_t page = 0;
  uint32_t run_low = 0, run_high = 0;
  auto look_up = [&](int key0) __attribute__((always_inline)) {      // (keys behind the last: its page, of which nothing is used)
    page = table[min(key0 + my_key, hi - 1) >> a.page_shift];
  };
  auto find_runs = [&](int key0) __attribute__((always_inline)) {
    const int slot = (key0 + my_key) & (a.page_size - 1);
    const uint64_t at = reinterpret_cast<uint64_t>(pools) + uint32_t(min(max(page, 0), a.num_pages - 1)) * page_bytes      // a bad table entry must not become a wild address
                        + uint32_t(lane < 16 ? slot * a.hd : my_dim + slot) * uint32_t(sizeof(E));
    run_low = uint32_t(at);
    run_high = uint32_t(at >> 32);
  };
  auto request = [&](int key0, int buffer) __attribute__((always_inline)) {
    const uint32_t at = lds_base + buffer * STAGE + 1024 * wave;
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      if (key0 + (wave + kWaves * u) / DT * GROUP >= hi) break;      // keys behind the last: their values are cleared, their scores masked
      auto start = [&](int from) { return uint64_t(uint32_t(__builtin_amdgcn_readlane(run_high, from))) << 32 | uint32_t(__builtin_amdgcn_readlane(run_low, from)); };
      if (whole || k_there[u]) lanes_to_lds(start(u), k_lane[u], at + 1024 * kWaves * u);
      if (whole || v_there[u]) lanes_to_lds(start(16 + u), v_lane, at + HALF + 1024 * kWaves * u);
    }
  };
  // Number by number, a piece at a time.
  auto copy = [&](int key0, int buffer) __attribute__((noinline)) {
    unsigned char* at = lds + buffer * STAGE;
    for (int i = threadIdx.x; i < HALF / 16; i += kThreads) {
      const int r = i / KC, c = place_in_row<KC>(r, i % KC), key = min(max(key0 + (kF32 ? r : swap23(r)), lo), hi - 1);
      const int index = key / a.page_size;
      const E* src = static_cast<const E*>(a.k_pool) + (page_of(index) * a.page_size + (key - index * a.page_size)) * a.hd + c * EPC;
      E e[EPC];
#pragma unroll
      for (int j = 0; j < EPC; ++j) e[j] = c * EPC + j < a.hd ? src[j] : from_float<E>(0.f);
      *reinterpret_cast<uint4*>(at + 16 * i) = *reinterpret_cast<uint4*>(e);
    }
    for (int i = threadIdx.x; i < HALF / 16; i += kThreads) {
      const int d = i / 64 % DT * 32 + i % 64 / 2, first = key0 + i / 64 / DT * GROUP + (i & 1) * EPC;
      E e[EPC];
#pragma unroll
      for (int j = 0; j < EPC; ++j) {
        const int key = min(max(first + j, lo), hi - 1), index = key / a.page_size;
        e[j] = d < a.hd ? static_cast<const E*>(a.v_pool)[(page_of(index) * a.hd + d) * a.page_size + (key - index * a.page_size)] : from_float<E>(0.f);
      }
      *reinterpret_cast<uint4*>(at + HALF + 16 * i) = *reinterpret_cast<uint4*>(e);
    }
  };
  // This thread's pieces of a stage's values.  Those of keys outside lo .. hi - 1 are cleared, whatever their slots hold (their weights are
  // zero, and zero times infinity is not), and so is what is not finite of keys that some rows see and others do not: that is added
  // at the end, to the rows that see it.
  bool left_out = false;
  auto look_at_values = [&](int key0, int buffer) __attribute__((always_inline)) {
#pragma unroll 1
    for (int i = threadIdx.x; i < HALF / 16; i += kThreads) {
      // RUNS: the thread's own loads, which have landed
      const int piece = i, key = key0 + piece / 64 / DT * GROUP + (piece & 1) * EPC;
      if (key >= lo && key + EPC <= min(hi, seen_by_all)) continue;
      uint4* place = reinterpret_cast<uint4*>(lds + buffer * STAGE + HALF + 16 * piece);
      uint32_t w[4] = {place->x, place->y, place->z, place->w};
#pragma unroll
      for (int j = 0; j < EPC; ++j) {
        const bool special = key + j >= seen_by_all && key + j < hi && not_finite<E>(w[j * 4 / EPC], j);
        left_out |= special;
        if (special || key + j < lo || key + j >= hi) w[j * 4 / EPC] &= ~bits_of<E>(j);
      }
      *place = make_uint4(w[0], w[1], w[2], w[3]);
    }
  };

  // ---- this lane's row
  uint4 q[STEPS];
  {
    const E* src = static_cast<const E*>(a.q) + size_t(token) * a.q_stride + size_t(head) * a.hd;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int d = (2 * s + lk) * EPC;
      if (RUNS) {
        q[s] = d < a.hd ? ldg128(src + d) : make_uint4(0, 0, 0, 0);
      } else {
        E e[EPC];
#pragma unroll
        for (int j = 0; j < EPC; ++j) e[j] = d + j < a.hd ? src[d + j] : from_float<E>(0.f);
        q[s] = *reinterpret_cast<uint4*>(e);
      }
    }
  }
  floatx16 o[DT];
  float m = kNothingYet, sums[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;

  uint32_t k_at[STEPS];      // where this lane's pieces of a tile's keys lie (tile 0; an odd tile's may lie otherwise, see below)
#pragma unroll
  for (int st = 0; st < STEPS; ++st) k_at[st] = 16 * (li * KC + place_in_row<KC>(li, 2 * st + lk));
  const uint32_t v_at = HALF + 32 * li + 16 * lk;
  const bool plain = a.cap == 0.f && a.scale2 > 0.f;      // the maximum of the scores is that of the products
  const float factor = plain ? a.scale2 : 1.f;

  if (RUNS) {
    look_up(first_key);
    find_runs(first_key);
    request(first_key, 0);
    look_up(first_key + KEYS);
  }
  int buffer = 0;
  for (int key0 = first_key; key0 < hi; key0 += KEYS, buffer ^= 1) {
    if (RUNS) asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
    else copy(key0, buffer);
    if (key0 < lo || key0 + KEYS > seen_by_all) look_at_values(key0, buffer);
    __syncthreads();
    const unsigned char* stage = lds + buffer * STAGE;
    bool asked = !RUNS || key0 + KEYS >= hi;
    auto ask = [&]() __attribute__((always_inline)) {      // the next stage, asked for while the first products run
      if (asked) return;
      asked = true;
      find_runs(key0 + KEYS);
      request(key0 + KEYS, buffer ^ 1);
      look_up(key0 + 2 * KEYS);
    };
    // N tiles of 32 keys, `shares` tiles apart, at once: their chains of dependent products and exponentials run side by side
    auto tiles = [&](auto count, int kt0) __attribute__((always_inline)) {
      constexpr int N = decltype(count)::value;
      floatx16 s[N];
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[n][r] = 0.f;
#pragma unroll
      for (int st = 0; st < STEPS; ++st)
#pragma unroll
        for (int n = 0; n < N; ++n) {      // (rows of eight pieces: 32 rows on, bit 2 of a piece's place is the other one)
          const int kt = kt0 + n * shares;
          const uint32_t at = (KC == 8 ? k_at[st] ^ ((kt & 1) << 6) : k_at[st]) + 32 * KC * 16 * kt;
          s[n] = piece_product(*reinterpret_cast<const uint4*>(stage + at), q[st], s[n], E());
        }
      ask();
      // A product's numbers may be read 12 wait states after its issue, of float32 18, and behind branches the compiler leaves fewer.
      __builtin_amdgcn_sched_barrier(0);
      if (kF32) asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 1");
      else asm volatile("s_nop 7\n\ts_nop 3");
      __builtin_amdgcn_sched_barrier(0);
      if (!plain) {
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[n][r] = a.cap > 0.f ? capped(s[n][r] * a.scale2, a.cap) : s[n][r] * a.scale2;
      }
      if (key0 + 32 * kt0 < lo || key0 + 32 * (kt0 + (N - 1) * shares) + 31 >= seen_by_all) {
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int key = key0 + 32 * (kt0 + n * shares) + (kF32 ? 8 * (r / 4) + 4 * lk + r % 4 : 16 * (r / 8) + 8 * lk + r % 8);
            if (key < lo || key > last) s[n][r] = -INFINITY;
          }
      }
      float tops[2] = {s[0][0], s[0][1]};
#pragma unroll
      for (int i = 2; i < 16 * N; i += 4) {
        tops[0] = largest(tops[0], s[i / 16][i % 16], s[(i + 1) / 16][(i + 1) % 16]);
        if (i + 3 < 16 * N) tops[1] = largest(tops[1], s[(i + 2) / 16][(i + 2) % 16], s[(i + 3) / 16][(i + 3) % 16]);
      }
      float top = larger(tops[0], tops[1]) * factor;
      if (__builtin_amdgcn_ballot_w64(top > m + kMaxMoves) != 0) {
        top = larger(top, other_half(top));
        const float next = top > m + kMaxMoves ? top : m, alpha = __builtin_amdgcn_exp2f(m - next);
        m = next;
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[i] *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
      }
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[n][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][r], factor, -m));
          sums[r % 4] += s[n][r];
        }
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int ps = 0; ps < PSTEPS; ++ps) {
          const uint4 w = weights_of(s[n], ps, E());
          const unsigned char* from = stage + v_at + ((kt0 + n * shares) * PSTEPS + ps) * HD * 32;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) o[dt] = piece_product(*reinterpret_cast<const uint4*>(from + 1024 * dt), w, o[dt], E());
        }
    };
    if (live) {
      int kt = share;
      constexpr bool kPairs = TILES > 1 && HD <= 128;
      if (kPairs)
        for (; kt + shares < TILES && key0 + 32 * (kt + shares) < hi; kt += 2 * shares) tiles(std::integral_constant<int, kPairs ? 2 : 1>(), kt);
      if (kt < TILES && key0 + 32 * kt < hi) tiles(std::integral_constant<int, 1>(), kt);
    }
    ask();
  }
  float l = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  l += other_half(l);

  // ---- waves that shared out the keys of the same rows join through LDS, half of them handing over to the other half, until one has all
  constexpr int PITCH = HD + 4;      // 16-byte places of a row's next one lie four banks on
  for (int half = shares >> 1; half > 0; half >>= 1) {
    __syncthreads();      // what lay here has been used
    float* buffer = reinterpret_cast<float*>(lds) + (((share & (half - 1)) << shift) + tile) * 32 * PITCH + li * PITCH;
    if (live && share >= half && share < 2 * half) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
          *reinterpret_cast<float4*>(buffer + 32 * dt + 2 * r + 4 * lk) = make_float4(o[dt][r], o[dt][r + 1], o[dt][r + 2], o[dt][r + 3]);
      if (lk == 0) { buffer[HD] = m; buffer[HD + 1] = l; }
    }
    __syncthreads();
    if (live && share < half) {
      const float m2 = buffer[HD], l2 = buffer[HD + 1], top = larger(m, m2);
      const float w1 = __builtin_amdgcn_exp2f(m - top), w2 = __builtin_amdgcn_exp2f(m2 - top);
      m = top;
      l = l * w1 + l2 * w2;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          const float4 b = *reinterpret_cast<const float4*>(buffer + 32 * dt + 2 * r + 4 * lk);
          o[dt][r] = o[dt][r] * w1 + b.x * w2;
          o[dt][r + 1] = o[dt][r + 1] * w1 + b.y * w2;
          o[dt][r + 2] = o[dt][r + 2] * w1 + b.z * w2;
          o[dt][r + 3] = o[dt][r + 3] * w1 + b.w * w2;
        }
    }
  }
  // (the pieces have been looked at by all threads; every thread comes here)
  if (own && seen_by_all < hi && __syncthreads_or(left_out)) {
    for (int key = max(seen_by_all, lo); key <= last; ++key) {
      const int index = key / a.page_size;
      const E* values = static_cast<const E*>(a.v_pool) + page_of(index) * a.hd * a.page_size + (key - index * a.page_size);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        __builtin_amdgcn_sched_barrier(0);      // (rare: few registers matter more than the loads' trips)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int d = 32 * dt + 8 * (r / 4) + 4 * lk + r % 4;
          const float v = d < a.hd ? to_float(values[size_t(d) * a.page_size]) : 0.f;
          if (!(fabsf(v) < INFINITY)) o[dt][r] += v;
        }
      }
    }
  }
  if (!live || share != 0 || !real) return;
  float* dst = a.part_o + (size_t(slot) * a.tokens * a.nq + place) * HD;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; r += 4)
      *reinterpret_cast<float4*>(dst + 32 * dt + 2 * r + 4 * lk) = make_float4(o[dt][r], o[dt][r + 1], o[dt][r + 2], o[dt][r + 3]);
  if (lk == 0) { ml[0] = m; ml[1] = l; }
}

// Joins the parts of the rows of one entry of the tile list (grid x), WAVES waves a row, rows dealt out over grid y.  Every lane of a wave
// looks at one part's statistics; HD / 4 lanes read a part's sums, so that the row's waves have 64 WAVES / (HD / 4) parts on their way at a time
// and four times that with the loads of four turns: one after the other, 33 parts of 640 rows of 128 took 14 us.
template <typename E, int HD, int WAVES>
__global__ __launch_bounds__(256) void attention_shared_join_kernel(SharedArgs a, E* __restrict__ out) {
  constexpr int LANES = HD / 4, AT_ONCE = 64 * WAVES / LANES, ROWS = 4 / WAVES, AHEAD = 4;
  __shared__ float4 s_sums[WAVES > 1 ? WAVES : 1][LANES];
  const int seq = a.tiles[2 * blockIdx.x], q_off = a.tiles[2 * blockIdx.x + 1];
  const int queries = min(kSharedTile, a.q_len[seq] - q_off), rows = queries * a.nq;
  const size_t first = size_t(a.q_start[seq] + q_off) * a.nq;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, in_row = threadIdx.x % (64 * WAVES);
  const int parts = a.prefix_splits + a.own_splits, dim = 4 * (in_row % LANES), turn = in_row / LANES;
  const size_t between = size_t(a.tokens) * a.nq;
  for (int r0 = blockIdx.y * ROWS; r0 < rows; r0 += gridDim.y * ROWS) {
    const int r = min(r0 + wave / WAVES, rows - 1);      // (a wave without a row goes along and writes nothing)
    const size_t place = first + r;
    float m = a.sinks ? a.sinks[r % a.nq] * kLog2E : kNothingYet, l = a.sinks && lane == 0 ? 1.f : 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p0 = 0; p0 < parts; p0 += 64) {
      float pm = kNothingYet, pl = 0.f;
      if (p0 + lane < parts) {
        const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + ((p0 + lane) * between + place) * 2);
        pm = ml.x;
        pl = ml.y;
      }
      const bool there = !(pm == kNothingYet && pl == 0.f);      // (a part that has seen nothing has not written its sums)
      float top = larger(m, pm);
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) top = larger(top, __shfl_xor(top, o, 64));
      const float before = __builtin_amdgcn_exp2f(m - top), w = there ? __builtin_amdgcn_exp2f(pm - top) : 0.f;
      m = top;
      l = l * before + (there ? pl * w : 0.f);
      acc.x *= before; acc.y *= before; acc.z *= before; acc.w *= before;
      const int n = min(64, parts - p0);
      for (int p = 0; p < n; p += AHEAD * AT_ONCE) {      // (all lanes walk: they hand each other the parts' weights)
        float4 v[AHEAD];
        float ws[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          const int mine = p + turn + i * AT_ONCE;
          ws[i] = __shfl(w, mine & 63, 64);
          const int seen = __shfl(int(there), mine & 63, 64);
          const bool read = mine < n && seen;
          v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (read) v[i] = *reinterpret_cast<const float4*>(a.part_o + ((p0 + mine) * between + place) * HD + dim);
          else ws[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) { acc.x += v[i].x * ws[i]; acc.y += v[i].y * ws[i]; acc.z += v[i].z * ws[i]; acc.w += v[i].w * ws[i]; }
      }
    }
    l = wave_sum(l);
#pragma unroll
    for (int o = LANES; o < 64; o <<= 1) {
      acc.x += __shfl_xor(acc.x, o, 64); acc.y += __shfl_xor(acc.y, o, 64); acc.z += __shfl_xor(acc.z, o, 64); acc.w += __shfl_xor(acc.w, o, 64);
    }
    if (WAVES > 1) {
      if (lane < LANES) s_sums[wave][lane] = acc;
      __syncthreads();
      if (wave == 0 && lane < LANES)
#pragma unroll
        for (int i = 1; i < WAVES; ++i) {
          const float4 v = s_sums[i][lane];
          acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
        }
      __syncthreads();
    }
    if (lane >= LANES || (WAVES > 1 ? wave != 0 : r0 + wave >= rows)) continue;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const float v[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (dim + j < a.hd) out[place * a.hd + dim + j] = from_float<E>(v[j]);
  }
}

int held_dims(int hd) { return hd <= 32 ? 32 : hd <= 64 ? 64 : hd <= 128 ? 128 : 256; }
int keys_of_stage(int dtype, int held) {
  const int bytes = held * (dtype == kF32 ? 4 : 2);
  return bytes <= 128 ? 128 : bytes <= 256 ? 64 : 32;
}

// Rows of heads, numbers of a token and keys, with a part's or a block's more, are counted in 32 bits.
bool shared_fits(int hd, int nq, int tokens, int max_ctx) { return int64_t(tokens) * nq <= 1 << 30 && int64_t(nq) * hd <= 1 << 30 && max_ctx <= 1 << 30; }

struct SharedPlan { int prefix_splits, prefix_keys, row_blocks, block_rows, own_splits, own_keys, own_rows; };

// How the work is cut: the shared keys of a block of rows into the number of parts with the least estimated time in microseconds.  A
// stage takes 1.35 alone on the chip and 0.85 more for every block that an XCD's CUs have on average (2.2 with one, 3.0 with two: measured with 44 to
// 484 blocks); units of a part and a key/value head go round the XCDs whole, so an XCD has the rows' blocks of some or of one unit more; behind two
// blocks a CU the rest waits.  A part costs what it writes and the joining launch reads.  A block of own keys counts for a quarter, as few rows share
// its waves' work.  Own keys come last and are cut into half as many stages, so that the end is even, and four at least; of float32, whose stages
// take four times as long, one (8 sequences of 3 queries behind 1,500 keys and 8 to 200 own: 15.8 us, with four 21.1).
// (64 sequences of 1 to 5 queries of 28 heads of 128 behind 8,192 keys, in all: 5, 7, 8, 9, 10, 11 parts 64.5, 57.5, 56.4, 62.4, 62.1, 65.0 us; 16 of
// one query of 40 heads behind 32,000: 25, 32, 48, 64 parts 43.2, 39.5, 38.2, 43.0.)
SharedPlan shared_plan(int dtype, int hd, int nq, int nkv, int tokens, int n_tiles, int prefix, int max_own) {
  SharedPlan p;
  const int G = nq / nkv, held = held_dims(hd), stage = keys_of_stage(dtype, held), rows = tokens * G;
  p.row_blocks = (rows + 127) / 128;
  p.block_rows = ((rows + p.row_blocks - 1) / p.row_blocks + 31) / 32 * 32;
  p.row_blocks = (rows + p.block_rows - 1) / p.block_rows;
  const int stages = (prefix + stage - 1) / stage;
  const int most = tokens - (n_tiles - 1) < kSharedTile ? tokens - (n_tiles - 1) : kSharedTile;      // every entry has a query
  p.own_rows = (most * G + 127) / 128;
  const double own_blocks = double(n_tiles) * ((tokens + n_tiles - 1) / n_tiles * G + 127) / 128 * nkv, part = double(tokens) * nq * held * 8.0 / 1.5e6;
  double best = 1.0e30;
  int chosen = 1;
  for (int splits = 1; splits <= 64 && splits <= stages; ++splits) {
    const int per = (stages + splits - 1) / splits;
    const int units = (splits * nkv + 7) / 8;      // of an XCD
    const double load = (double(units) * p.row_blocks + own_blocks / 32.0) / 32.0;
    const double time = per * (1.35 + 0.85 * load) * (load > 2.0 ? load / 2.0 : 1.0) + splits * part;
    if (time < best) { best = time; chosen = per; }
  }
  p.prefix_keys = chosen * stage;
  p.prefix_splits = (stages + chosen - 1) / chosen;
  const int least = dtype == kF32 ? 1 : 4, own_stages = (max_own + stage - 1) / stage, of_64 = (own_stages + 63) / 64;      // 64 parts at most, as of the shared keys
  const int own = chosen / 2 > least ? chosen / 2 : least;
  p.own_keys = (own > of_64 ? own : of_64) * stage;
  p.own_splits = (max_own + p.own_keys - 1) / p.own_keys;
  return p;
}

template <typename E, int HD, bool RUNS> int launch_shared(hipStream_t s, const SharedArgs& a, int blocks, dim3 join_grid, void* out) {
  constexpr int bytes = 4 * stage_keys<E, HD>() * HD * int(sizeof(E)), join = kWaves / 2 * 32 * (HD + 4) * 4;      // two stages; tiles handed over
  constexpr int lds = bytes > join ? bytes : join;
  static bool raised[64] = {};      // by device: the attribute is the device's copy of the kernel's
  int device = 0;
  hipError_t e = hipGetDevice(&device);
  if (e == hipSuccess && (device < 0 || device >= 64 || !raised[device])) {
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(attention_shared_kernel<E, HD, RUNS>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e == hipSuccess && device >= 0 && device < 64) raised[device] = true;
  }
  if (e != hipSuccess) {
    set_error("sp_attention_shared: cannot raise the LDS limit: %s", hipGetErrorString(e));
    return 1;
  }
  attention_shared_kernel<E, HD, RUNS><<<blocks, 64 * kWaves, lds, s>>>(a);
  // few parts: a wave has them all on their way at once; with more, four waves share a row's, unless there are rows enough to fill the chip
  // with waves (5,404 rows of 12 parts of 128: four waves 15 us)
  if (a.prefix_splits + a.own_splits <= 4 * (256 / HD) || int64_t(a.tokens) * a.nq >= 4096) attention_shared_join_kernel<E, HD, 1><<<join_grid, 256, 0, s>>>(a, static_cast<E*>(out));
  else attention_shared_join_kernel<E, HD, 4><<<dim3(join_grid.x, 4 * join_grid.y), 256, 0, s>>>(a, static_cast<E*>(out));
  return check_launch("sp_attention_shared");
}
template <typename E> int launch_shared_of(hipStream_t s, const SharedArgs& a, int blocks, int held, bool runs, dim3 join_grid, void* out) {
  switch (held) {
    case 32: return runs ? launch_shared<E, 32, true>(s, a, blocks, join_grid, out) : launch_shared<E, 32, false>(s, a, blocks, join_grid, out);
    case 64: return runs ? launch_shared<E, 64, true>(s, a, blocks, join_grid, out) : launch_shared<E, 64, false>(s, a, blocks, join_grid, out);
    case 128: return runs ? launch_shared<E, 128, true>(s, a, blocks, join_grid, out) : launch_shared<E, 128, false>(s, a, blocks, join_grid, out);
    default: return runs ? launch_shared<E, 256, true>(s, a, blocks, join_grid, out) : launch_shared<E, 256, false>(s, a, blocks, join_grid, out);
  }
}

}  // namespace

}  // namespace sprout

using namespace sprout;

extern "C" int64_t sp_attention_shared_workspace_floats(int dtype, int hd, int nq, int nkv, int tokens, int n_tiles, int prefix, int max_ctx) {
  if (hd <= 0 || hd > 256 || nkv <= 0 || nq <= 0 || nq % nkv || tokens <= 0 || n_tiles <= 0 || n_tiles > tokens || prefix < 0 || max_ctx <= prefix ||
      !shared_fits(hd, nq, tokens, max_ctx)) return 0;
  const SharedPlan p = shared_plan(dtype, hd, nq, nkv, tokens, n_tiles, prefix, max_ctx - prefix);
  return (int64_t(p.prefix_splits) + p.own_splits) * tokens * nq * (held_dims(hd) + 2);
}

extern "C" int sp_attention_shared(void* stream, int dtype, const void* q, int q_stride, const void* k_pool, const void* v_pool,
                                   const int32_t* block_tables, int max_blocks, const int32_t* prefix_table, int prefix,
                                   const int32_t* q_start, const int32_t* q_len, const int32_t* ctx_len, const int32_t* tiles, int n_tiles,
                                   int max_ctx, int tokens, float* workspace, int64_t workspace_floats, void* out, int nq, int nkv, int hd,
                                   int page_size, int num_pages, float scale, float softcap, const float* sinks) {
  SP_REQUIRE(dtype == kF32 || dtype == kBF16, "sp_attention_shared: unsupported dtype %d", dtype);
  SP_REQUIRE(nq > 0 && nkv > 0 && nq % nkv == 0, "sp_attention_shared: %d query heads do not divide into %d groups", nq, nkv);
  SP_REQUIRE(hd > 0 && hd <= 256, "sp_attention_shared: head size %d is outside 1..256", hd);
  SP_REQUIRE(page_size > 0 && num_pages > 0 && max_blocks > 0 && int64_t(max_blocks) * page_size < int64_t(1) << 31, "sp_attention_shared: bad cache geometry");
  SP_REQUIRE(n_tiles >= 0 && tokens >= n_tiles, "sp_attention_shared: %d tiles of queries for %d rows", n_tiles, tokens);
  if (n_tiles == 0) return 0;
  SP_REQUIRE(q && k_pool && v_pool && block_tables && q_start && q_len && ctx_len && tiles && out && (prefix_table || prefix == 0),
             "sp_attention_shared: null operand");
  SP_REQUIRE(shared_fits(hd, nq, tokens, max_ctx), "sp_attention_shared: %d rows of %d heads of %d with contexts of up to %d are more than indexes hold", tokens, nq, hd, max_ctx);
  SP_REQUIRE(q_stride >= nq * hd, "sp_attention_shared: q row stride %d is smaller than %d", q_stride, nq * hd);
  SP_REQUIRE(prefix >= 0 && max_ctx > prefix && int64_t(max_ctx) <= int64_t(max_blocks) * page_size,
             "sp_attention_shared: a prefix of %d and contexts of up to %d do not fit %d pages of %d", prefix, max_ctx, max_blocks, page_size);
  SP_REQUIRE(softcap >= 0.f && softcap < INFINITY, "sp_attention_shared: a cap that is negative or not finite");
  const SharedPlan p = shared_plan(dtype, hd, nq, nkv, tokens, n_tiles, prefix, max_ctx - prefix);
  const int held = held_dims(hd);
  const int64_t need = sp_attention_shared_workspace_floats(dtype, hd, nq, nkv, tokens, n_tiles, prefix, max_ctx);
  SP_REQUIRE(workspace && workspace_floats >= need, "sp_attention_shared: workspace of %lld floats is smaller than the %lld needed",
             (long long)workspace_floats, (long long)need);
  const int64_t rows = int64_t(tokens) * nq, parts = int64_t(p.prefix_splits) + p.own_splits;
  const int64_t blocks = (int64_t(p.prefix_splits) * nkv + 7) / 8 * 8 * p.row_blocks + int64_t(p.own_splits) * n_tiles * p.own_rows * nkv;
  SP_REQUIRE(blocks < 1 << 24, "sp_attention_shared: %lld blocks are more than a launch takes", (long long)blocks);      // less than 2^32 threads
  SharedArgs a;
  a.q = q; a.k_pool = k_pool; a.v_pool = v_pool;
  a.block_tables = block_tables; a.prefix_table = prefix_table; a.q_start = q_start; a.q_len = q_len; a.ctx_len = ctx_len; a.tiles = tiles;
  a.part_o = workspace;
  a.part_ml = workspace + parts * rows * held;
  a.sinks = sinks;
  a.q_stride = q_stride; a.max_blocks = max_blocks; a.prefix = prefix; a.tokens = tokens; a.n_tiles = n_tiles;
  a.nq = nq; a.nkv = nkv; a.hd = hd; a.page_size = page_size; a.num_pages = num_pages;
  a.prefix_splits = p.prefix_splits; a.prefix_keys = p.prefix_keys; a.row_blocks = p.row_blocks; a.block_rows = p.block_rows;
  a.own_splits = p.own_splits; a.own_keys = p.own_keys; a.own_rows = p.own_rows;
  a.scale2 = softcap > 0.f ? 2.f * kLog2E * scale / softcap : scale * kLog2E;
  a.cap = softcap;
  const int epc = dtype == kF32 ? 4 : 8;
  const uintptr_t bases = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool);
  a.page_shift = 0;
  while ((1 << a.page_shift) < page_size && a.page_shift < 30) ++a.page_shift;
  const bool runs = hd % epc == 0 && page_size >= 16 && (1 << a.page_shift) == page_size && page_size <= 4096 && q_stride % epc == 0 && bases % 16 == 0;
  // blocks for the rows that an entry has on average (four rows a block); those of longer entries are walked in turns
  const int64_t in_entry = (tokens + n_tiles - 1) / n_tiles < kSharedTile ? (tokens + n_tiles - 1) / n_tiles : kSharedTile, of_four = (in_entry * nq + 3) / 4;
  const dim3 join_grid(n_tiles, of_four < 16383 ? of_four : 16383);      // (times four below 65,536, the most along y)
  hipStream_t s = (hipStream_t)stream;
  return dtype == kF32 ? launch_shared_of<float>(s, a, int(blocks), held, runs, join_grid, out)
                       : launch_shared_of<bf16_t>(s, a, int(blocks), held, runs, join_grid, out);
}
