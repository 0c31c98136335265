// Attention of a batch whose sequences begin with the same keys: the shared keys are read once for all rows, then each sequence's own.
//
//   s = scale q . k (capped: c tanh(s / c)),  w = exp(s - m),  o = sum w v / sum w     over the keys up to the query's position.
// A softmax over disjoint ranges of keys joins: with each range's maximum m_i, l_i = sum exp(s - m_i) and o_i = sum exp(s - m_i) v,
// m = max m_i, l = sum l_i exp(m_i - m), o = sum o_i exp(m_i - m) / l.  So the work is cut into items, each some rows by some keys of one
// key/value head, that leave (m, l, o) in the workspace in float32; a second launch joins a row's parts in a fixed order.
// A row is a token and a head of the group: rows of one key/value head are numbered token by token, so that the rows of all sequences
// multiply the shared keys in one product, and a sequence's own keys are met by its own rows alone.
//
// An item is a block of four waves: up to 128 rows in tiles of 32, a wave a tile; with fewer rows the waves share out the keys of
// a stage and join at the end.  Keys and values go through LDS in stages, loaded into registers while the stage before is used:
//   S^T[key, row] = K . Q^T,   O^T[dim, row] += V^T . P^T       32x32 matrix instructions, queries, sums and statistics in registers.
// The product S^T leaves a lane 16 keys of one row.  bfloat16: key rows lie in LDS with bits 2 and 3 of their number swapped, which
// makes a lane's keys two runs of eight: what the second product takes as its operand.  float32: runs of four, as the float32
// instruction takes them; nothing is rounded before the result.
// Weights are rounded to bfloat16 for the product with the values (half a step each); the sum of the weights is of the unrounded ones.
#include <type_traits>

#include "mfma.h"
#include "sprout_hip.h"

namespace sprout {

namespace {

constexpr float kLog2E = 1.4426950408889634f;
constexpr float kNothingYet = -1.0e30f;      // running maximum before any key: finite, so that no inf - inf arises
constexpr float kMaxMoves = 8.0f;            // the running maximum follows the true one when that lies further above it (log2): until
                                             // then weights reach 2^8 at most, which float32 and bfloat16 hold as well as 1
constexpr int kSharedTable = 1024;           // page numbers of an item kept in LDS
constexpr int kSharedTile = 16;              // queries of one entry of the tile list

struct SharedArgs {
  const void *q, *k_pool, *v_pool;
  const int32_t *block_tables, *prefix_table, *q_start, *q_len, *ctx_len, *tiles;
  float *part_o, *part_ml;
  const float* sinks;
  int q_stride, max_blocks, prefix, tokens, n_tiles, nq, nkv, hd, page_size, num_pages;
  int prefix_splits, prefix_keys, row_blocks, block_rows;      // shared keys: parts, keys of each, blocks of rows, rows of each
  int own_splits, own_keys, own_rows;                          // own keys: parts, keys of each, blocks of 128 rows of an entry
  float scale2, cap;                                           // scale in log2 units; the cap (0: none), of the scale without them
};

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
__device__ __forceinline__ float other_half(float x) {      // lane ^ 32's
  const unsigned u = __float_as_uint(x);
  const auto f = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float((threadIdx.x & 32) ? f[0] : f[1]);
}

template <typename E> __device__ __forceinline__ bool any_not_finite(uint4 v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (std::is_same<E, float>::value) bad |= (w[i] & 0x7f800000u) == 0x7f800000u;
    else bad |= (w[i] & 0x7f80u) == 0x7f80u || (w[i] & 0x7f800000u) == 0x7f800000u;
  }
  return bad;
}
// The piece with what is not finite taken out (kind 0), or 1 where a number is NaN (1), +infinity (2), -infinity (3) and 0 elsewhere.
template <typename E> __device__ __forceinline__ uint4 only(uint4 v, int kind) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (std::is_same<E, float>::value) {
      const uint32_t m = w[i] & 0x7fffffffu;
      const int what = m < 0x7f800000u ? 0 : m > 0x7f800000u ? 1 : (w[i] >> 31) ? 3 : 2;
      w[i] = kind == 0 ? (what ? 0u : w[i]) : what == kind ? 0x3f800000u : 0u;
    } else {
      uint32_t out = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t x = (w[i] >> (16 * h)) & 0xffffu, m = x & 0x7fffu;
        const int what = m < 0x7f80u ? 0 : m > 0x7f80u ? 1 : (x >> 15) ? 3 : 2;
        out |= (kind == 0 ? (what ? 0u : x) : what == kind ? 0x3f80u : 0u) << (16 * h);
      }
      w[i] = out;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
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

// Keys of a stage: 64 KB of keys and values at most.
template <typename E, int HD> constexpr int stage_keys() { return HD * int(sizeof(E)) <= 256 ? 128 : HD * int(sizeof(E)) <= 512 ? 64 : 32; }

// E: the numbers' type, HD: dimensions held (the head's size or the next one up, zeros behind it), VEC: pieces of 16 bytes can be loaded.
template <typename E, int HD, bool VEC>
__global__ __launch_bounds__(256, HD * sizeof(E) <= 256 ? 2 : 1) void attention_shared_kernel(SharedArgs a) {
  constexpr int EPC = Numbers<E>::kChunk, KEYS = stage_keys<E, HD>(), KC = HD / EPC, VC = KEYS / EPC, TILES = KEYS / 32;
  constexpr int PIECES = KEYS * HD / EPC / 256, DT = HD / 32, STEPS = HD / (2 * EPC), PSTEPS = 32 / (2 * EPC);
  constexpr bool kF32 = std::is_same<E, float>::value;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  unsigned char *lds_k = lds, *lds_v = lds + KEYS * HD * sizeof(E);
  int32_t* s_table = reinterpret_cast<int32_t*>(lds + 2 * KEYS * HD * sizeof(E));

  // ---- which item: rows first_row .. + rows of key/value head g, keys lo .. hi - 1, part `slot`
  const int G = a.nq / a.nkv;
  const int prefix_items = a.prefix_splits * a.row_blocks * a.nkv;
  int g, first_row, rows, lo, hi, slot, seq = -1, first_pos = 0, first_token = 0;
  const int32_t* table;
  if (int(blockIdx.x) < prefix_items) {
    const int rb = blockIdx.x % a.row_blocks, rest = blockIdx.x / a.row_blocks;
    g = rest % a.nkv;
    slot = rest / a.nkv;
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
    seq = a.tiles[2 * entry];
    const int q_off = a.tiles[2 * entry + 1], len = a.q_len[seq], ctx = a.ctx_len[seq];
    const int queries = min(kSharedTile, len - q_off);
    first_token = a.q_start[seq] + q_off;
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
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, li = lane & 31, lk = lane >> 5;
  const int row_tiles = (rows + 31) / 32;
  const int shift = row_tiles == 1 ? 0 : row_tiles == 2 ? 1 : 2;      // 1, 2 or 4 waves side by side along the rows
  const int tile = wave & ((1 << shift) - 1), share = wave >> shift, shares = 4 >> shift;
  const bool live = tile < row_tiles;
  const int row = first_row + min(32 * tile + li, rows - 1), token = row / G, head = g * G + (row - token * G);
  const size_t place = size_t(token) * a.nq + head;
  const bool real = 32 * tile + li < rows;
  float* ml = a.part_ml + (size_t(slot) * a.tokens * a.nq + place) * 2;
  if (hi <= lo) {      // own keys that end before this part: said to the joining launch, which reads every part's statistics
    if (live && share == 0 && real && lk == 0) { ml[0] = kNothingYet; ml[1] = 0.f; }
    return;
  }

  // ---- page numbers
  const int first_key = VEC ? lo / EPC * EPC : lo, first_page = first_key / a.page_size, pages = (hi - 1) / a.page_size - first_page + 1;
  const bool in_lds = pages <= kSharedTable;
  if (in_lds)
    for (int i = threadIdx.x; i < pages; i += 256) s_table[i] = table[first_page + i];
  __syncthreads();
  auto page_at = [&](int key, int& offset) __attribute__((always_inline)) {
    const int index = key / a.page_size;
    offset = key - index * a.page_size;
    const int page = in_lds ? s_table[index - first_page] : table[index];
    return size_t(min(max(page, 0), a.num_pages - 1)) * a.nkv + g;      // a bad table entry must not become a wild address
  };

  // ---- a stage's way: memory -> registers -> LDS
  uint4 kr[PIECES], vr[PIECES];
  auto fetch = [&](int key0) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < PIECES; ++u) {
      const int i = threadIdx.x + 256 * u, r = i / KC, c = place_in_row<KC>(r, i % KC);
      const int key = min(key0 + (kF32 ? r : swap23(r)), hi - 1);
      int at;
      const size_t page = page_at(key, at);
      const E* src = static_cast<const E*>(a.k_pool) + (page * a.page_size + at) * a.hd + c * EPC;
      if (VEC) {
        kr[u] = c * EPC < a.hd ? ldg128(src) : make_uint4(0, 0, 0, 0);
      } else {
        E e[EPC];
#pragma unroll
        for (int j = 0; j < EPC; ++j) e[j] = c * EPC + j < a.hd ? src[j] : from_float<E>(0.f);
        kr[u] = *reinterpret_cast<uint4*>(e);
      }
    }
#pragma unroll
    for (int u = 0; u < PIECES; ++u) {
      const int i = threadIdx.x + 256 * u, d = i / VC, c = place_in_row<VC>(d, i % VC);
      if (VEC) {
        int at;
        const size_t page = page_at(min(key0 + c * EPC, (hi - 1) / EPC * EPC), at);
        vr[u] = d < a.hd ? ldg128(static_cast<const E*>(a.v_pool) + (page * a.hd + d) * a.page_size + at) : make_uint4(0, 0, 0, 0);
      } else {
        E e[EPC];
#pragma unroll
        for (int j = 0; j < EPC; ++j) {
          int at;
          const size_t page = page_at(min(key0 + c * EPC + j, hi - 1), at);
          e[j] = d < a.hd ? static_cast<const E*>(a.v_pool)[(page * a.hd + d) * a.page_size + at] : from_float<E>(0.f);
        }
        vr[u] = *reinterpret_cast<uint4*>(e);
      }
    }
  };
  // Values of keys outside lo .. hi - 1 are cleared, whatever their slots hold: their weights are zero, and zero times infinity is not.
  auto to_lds = [&](int key0) __attribute__((always_inline)) {
    const bool ends = key0 < lo || key0 + KEYS > hi;
    bool bad = false;
#pragma unroll
    for (int u = 0; u < PIECES; ++u) *reinterpret_cast<uint4*>(lds_k + 16 * (threadIdx.x + 256 * u)) = kr[u];
#pragma unroll
    for (int u = 0; u < PIECES; ++u) {
      const int i = threadIdx.x + 256 * u, key = key0 + place_in_row<VC>(i / VC, i % VC) * EPC;
      if (ends) {
        uint32_t w[4] = {vr[u].x, vr[u].y, vr[u].z, vr[u].w};
#pragma unroll
        for (int j = 0; j < EPC; ++j)
          if (key + j < lo || key + j >= hi) w[j * 4 / EPC] &= kF32 ? 0u : (j & 1) ? 0x0000ffffu : 0xffff0000u;
        vr[u] = make_uint4(w[0], w[1], w[2], w[3]);
      }
      if (own) bad |= any_not_finite<E>(vr[u]);
      *reinterpret_cast<uint4*>(lds_v + 16 * i) = vr[u];
    }
    return bad;
  };

  // ---- this lane's row
  uint4 q[STEPS];
  {
    const E* src = static_cast<const E*>(a.q) + size_t(token) * a.q_stride + size_t(head) * a.hd;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int d = (2 * s + lk) * EPC;
      if (VEC) {
        q[s] = d < a.hd ? ldg128(src + d) : make_uint4(0, 0, 0, 0);
      } else {
        E e[EPC];
#pragma unroll
        for (int j = 0; j < EPC; ++j) e[j] = d + j < a.hd ? src[d + j] : from_float<E>(0.f);
        q[s] = *reinterpret_cast<uint4*>(e);
      }
    }
  }
  const int last = own ? min(first_pos + token - first_token, hi - 1) : hi - 1;      // the last key that the row sees
  const int seen_by_all = own ? min(first_pos + 1, hi) : hi;                          // keys before this one are seen by every row
  floatx16 o[DT];
  float m = kNothingYet, l = 0.f;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;

  fetch(first_key);
  for (int key0 = first_key; key0 < hi; key0 += KEYS) {
    if (key0 > first_key) __syncthreads();      // the stage before has been used
    const bool bad = to_lds(key0);
    // A value that is not finite must stay with the rows that see its key: rows that do not have weight zero for it
    const bool careful = own && key0 + KEYS > seen_by_all ? __syncthreads_or(bad) != 0 : (__syncthreads(), false);
    if (key0 + KEYS < hi) fetch(key0 + KEYS);
    if (!live) continue;
    for (int kt = share; kt < TILES; kt += shares) {
      const int first = key0 + 32 * kt;
      if (first >= hi) break;
      floatx16 s;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
      for (int st = 0; st < STEPS; ++st) {
        const int kr_row = 32 * kt + li;
        s = piece_product(*reinterpret_cast<const uint4*>(lds_k + 16 * (kr_row * KC + place_in_row<KC>(kr_row, 2 * st + lk))), q[st], s, E());
      }
      if (a.cap > 0.f) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = a.cap * kLog2E * tanhf(s[r] * a.scale2);
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= a.scale2;
      }
      if (first < lo || first + 31 >= seen_by_all) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = first + (kF32 ? 8 * (r / 4) + 4 * lk + r % 4 : 16 * (r / 8) + 8 * lk + r % 8);
          if (key < lo || key > last) s[r] = -INFINITY;
        }
      }
      float top = s[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) top = larger(top, s[r]);
      if (__builtin_amdgcn_ballot_w64(top > m + kMaxMoves) != 0) {
        top = larger(top, other_half(top));
        const float next = top > m + kMaxMoves ? top : m, alpha = __builtin_amdgcn_exp2f(m - next);
        m = next;
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = __builtin_amdgcn_exp2f(s[r] - m);
        l += s[r];
      }
#pragma unroll
      for (int ps = 0; ps < PSTEPS; ++ps) {
        const uint4 w = weights_of(s, ps, E());
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const int d = 32 * dt + li;
          const uint4 v = *reinterpret_cast<const uint4*>(lds_v + 16 * (d * VC + place_in_row<VC>(d, 32 * kt / EPC + 2 * ps + lk)));
          o[dt] = piece_product(careful ? only<E>(v, 0) : v, w, o[dt], E());
        }
      }
      if (careful) {      // how many of what a row sees is NaN, +infinity, -infinity, dimension by dimension
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = first + (kF32 ? 8 * (r / 4) + 4 * lk + r % 4 : 16 * (r / 8) + 8 * lk + r % 8);
          s[r] = key < lo || key > last ? 0.f : 1.f;
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          for (int kind = 1; kind <= 3; ++kind) {
            const float special = kind == 1 ? NAN : kind == 2 ? INFINITY : -INFINITY;
            floatx16 n;
#pragma unroll
            for (int r = 0; r < 16; ++r) n[r] = 0.f;
#pragma unroll
            for (int ps = 0; ps < PSTEPS; ++ps) {
              const int d = 32 * dt + li;
              const uint4 v = *reinterpret_cast<const uint4*>(lds_v + 16 * (d * VC + place_in_row<VC>(d, 32 * kt / EPC + 2 * ps + lk)));
              n = piece_product(only<E>(v, kind), weights_of(s, ps, E()), n, E());
            }
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (n[r] > 0.f) o[dt][r] += special;
          }
      }
    }
  }
  l += other_half(l);

  // ---- waves that shared out the keys of the same rows join through LDS, the first wave last
  if (shares > 1) {
    constexpr int PITCH = HD + 4;      // 16-byte places of a row's next one lie four banks on
    float* mine = reinterpret_cast<float*>(lds) + size_t(li) * PITCH;
    for (int from = 1; from < shares; ++from) {
      __syncthreads();      // what lay here has been used
      float* buffer = mine + size_t(tile) * 32 * PITCH;
      if (live && share == from) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int r = 0; r < 16; r += 4)
            *reinterpret_cast<float4*>(buffer + 32 * dt + 2 * r + 4 * lk) = make_float4(o[dt][r], o[dt][r + 1], o[dt][r + 2], o[dt][r + 3]);
        if (lk == 0) { buffer[HD] = m; buffer[HD + 1] = l; }
      }
      __syncthreads();
      if (live && share == 0) {
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

// Joins the parts of the rows of one entry of the tile list (grid x), a wave a row, rows dealt out over grid y.
template <typename E>
__global__ __launch_bounds__(256) void attention_shared_join_kernel(SharedArgs a, E* __restrict__ out, int held) {
  const int seq = a.tiles[2 * blockIdx.x], q_off = a.tiles[2 * blockIdx.x + 1];
  const int queries = min(kSharedTile, a.q_len[seq] - q_off);
  const size_t first = size_t(a.q_start[seq] + q_off) * a.nq;
  const int lane = threadIdx.x & 63, parts = a.prefix_splits + a.own_splits;
  const size_t between = size_t(a.tokens) * a.nq;
  for (int r = blockIdx.y * 4 + (threadIdx.x >> 6); r < queries * a.nq; r += gridDim.y * 4) {
    const size_t place = first + r;
    const float sink = a.sinks ? a.sinks[r % a.nq] * kLog2E : 0.f;
    float m = a.sinks ? sink : kNothingYet;
    for (int p = 0; p < parts; ++p) m = larger(m, a.part_ml[(p * between + place) * 2]);
    float l = a.sinks ? __builtin_amdgcn_exp2f(sink - m) : 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p = 0; p < parts; ++p) {
      const float pm = a.part_ml[(p * between + place) * 2], pl = a.part_ml[(p * between + place) * 2 + 1];
      if (pm == kNothingYet && pl == 0.f) continue;      // nothing seen there (its sums have not been written)
      const float w = __builtin_amdgcn_exp2f(pm - m);
      l += pl * w;
      if (4 * lane < held) {
        const float4 v = *reinterpret_cast<const float4*>(a.part_o + (p * between + place) * held + 4 * lane);
        acc.x += v.x * w; acc.y += v.y * w; acc.z += v.z * w; acc.w += v.w * w;
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const float v[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (4 * lane + j < a.hd) out[place * a.hd + 4 * lane + j] = from_float<E>(v[j]);
  }
}

int held_dims(int hd) { return hd <= 32 ? 32 : hd <= 64 ? 64 : hd <= 96 ? 96 : hd <= 128 ? 128 : hd <= 192 ? 192 : 256; }
int keys_of_stage(int dtype, int held) {
  const int bytes = held * (dtype == kF32 ? 4 : 2);
  return bytes <= 256 ? 128 : bytes <= 512 ? 64 : 32;
}

struct SharedPlan { int prefix_splits, prefix_keys, row_blocks, block_rows, own_splits, own_keys, own_rows; };

// How the work is cut: shared keys into as many parts as give the chip two blocks a CU, own keys into parts of 512.
SharedPlan shared_plan(int dtype, int hd, int nq, int nkv, int tokens, int n_tiles, int prefix, int max_own) {
  SharedPlan p;
  const int G = nq / nkv, held = held_dims(hd), stage = keys_of_stage(dtype, held), rows = tokens * G;
  p.row_blocks = (rows + 127) / 128;
  p.block_rows = ((rows + p.row_blocks - 1) / p.row_blocks + 31) / 32 * 32;
  p.row_blocks = (rows + p.block_rows - 1) / p.block_rows;
  const int stages = (prefix + stage - 1) / stage, blocks = p.row_blocks * nkv;
  const int want = (512 + blocks - 1) / blocks, per = stages > 0 ? (stages + (want < stages ? want : stages) - 1) / (want < stages ? want : stages) : 1;
  p.prefix_keys = per * stage;
  p.prefix_splits = (stages + per - 1) / per;
  p.own_keys = 512;
  p.own_splits = (max_own + p.own_keys - 1) / p.own_keys;
  const int most = tokens - (n_tiles - 1) < kSharedTile ? tokens - (n_tiles - 1) : kSharedTile;      // every entry has a query
  p.own_rows = (most * G + 127) / 128;
  return p;
}

template <typename E, int HD, bool VEC> int launch_shared(hipStream_t s, const SharedArgs& a, int blocks) {
  constexpr int bytes = 2 * stage_keys<E, HD>() * HD * int(sizeof(E));
  constexpr int join = 2 * 32 * (HD + 4) * 4;      // two tiles of rows handed over at a time
  const int lds = (bytes > join ? bytes : join) + 4 * kSharedTable;
  static bool raised[64] = {};      // by device: the attribute is the device's copy of the kernel's
  int device = 0;
  hipError_t e = hipGetDevice(&device);
  if (e == hipSuccess && (device < 0 || device >= 64 || !raised[device])) {
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(attention_shared_kernel<E, HD, VEC>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e == hipSuccess && device >= 0 && device < 64) raised[device] = true;
  }
  if (e != hipSuccess) {
    set_error("sp_attention_shared: cannot raise the LDS limit: %s", hipGetErrorString(e));
    return 1;
  }
  attention_shared_kernel<E, HD, VEC><<<blocks, 256, lds, s>>>(a);
  return check_launch("sp_attention_shared");
}
template <typename E, bool VEC> int launch_shared_of(hipStream_t s, const SharedArgs& a, int blocks, int held) {
  switch (held) {
    case 32: return launch_shared<E, 32, VEC>(s, a, blocks);
    case 64: return launch_shared<E, 64, VEC>(s, a, blocks);
    case 96: return launch_shared<E, 96, VEC>(s, a, blocks);
    case 128: return launch_shared<E, 128, VEC>(s, a, blocks);
    case 192: return launch_shared<E, 192, VEC>(s, a, blocks);
    default: return launch_shared<E, 256, VEC>(s, a, blocks);
  }
}

}  // namespace

}  // namespace sprout

using namespace sprout;

extern "C" int64_t sp_attention_shared_workspace_floats(int dtype, int hd, int nq, int nkv, int tokens, int n_tiles, int prefix, int max_ctx) {
  if (hd <= 0 || hd > 256 || nkv <= 0 || nq <= 0 || nq % nkv || tokens <= 0 || n_tiles <= 0 || n_tiles > tokens || prefix < 0 || max_ctx <= prefix) return 0;
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
  SP_REQUIRE(page_size > 0 && num_pages > 0 && max_blocks > 0, "sp_attention_shared: bad cache geometry");
  SP_REQUIRE(n_tiles >= 0 && tokens >= n_tiles, "sp_attention_shared: %d tiles of queries for %d rows", n_tiles, tokens);
  if (n_tiles == 0) return 0;
  SP_REQUIRE(q && k_pool && v_pool && block_tables && q_start && q_len && ctx_len && tiles && out && (prefix_table || prefix == 0),
             "sp_attention_shared: null operand");
  SP_REQUIRE(q_stride >= nq * hd, "sp_attention_shared: q row stride %d is smaller than %d", q_stride, nq * hd);
  SP_REQUIRE(prefix >= 0 && max_ctx > prefix && int64_t(max_ctx) <= int64_t(max_blocks) * page_size,
             "sp_attention_shared: a prefix of %d and contexts of up to %d do not fit %d pages of %d", prefix, max_ctx, max_blocks, page_size);
  SP_REQUIRE(softcap >= 0.f, "sp_attention_shared: negative cap");
  const SharedPlan p = shared_plan(dtype, hd, nq, nkv, tokens, n_tiles, prefix, max_ctx - prefix);
  const int held = held_dims(hd);
  const int64_t need = sp_attention_shared_workspace_floats(dtype, hd, nq, nkv, tokens, n_tiles, prefix, max_ctx);
  SP_REQUIRE(workspace && workspace_floats >= need, "sp_attention_shared: workspace of %lld floats is smaller than the %lld needed",
             (long long)workspace_floats, (long long)need);
  const int64_t rows = int64_t(tokens) * nq, parts = int64_t(p.prefix_splits) + p.own_splits;
  const int64_t blocks = int64_t(p.prefix_splits) * p.row_blocks * nkv + int64_t(p.own_splits) * n_tiles * p.own_rows * nkv;
  SP_REQUIRE(blocks < (int64_t(1) << 31), "sp_attention_shared: too many blocks");
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
  a.scale2 = softcap > 0.f ? scale / softcap : scale * kLog2E;
  a.cap = softcap;
  const int epc = dtype == kF32 ? 4 : 8;
  const uintptr_t bases = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool);
  const bool vec = hd % epc == 0 && page_size % epc == 0 && q_stride % epc == 0 && bases % 16 == 0;
  hipStream_t s = (hipStream_t)stream;
  const int rc = dtype == kF32 ? (vec ? launch_shared_of<float, true>(s, a, int(blocks), held) : launch_shared_of<float, false>(s, a, int(blocks), held))
                               : (vec ? launch_shared_of<bf16_t, true>(s, a, int(blocks), held) : launch_shared_of<bf16_t, false>(s, a, int(blocks), held));
  if (rc) return rc;
  const int most = tokens - (n_tiles - 1) < kSharedTile ? tokens - (n_tiles - 1) : kSharedTile;
  const int want = (most * nq + 3) / 4, cap = 4096 / n_tiles + 1;
  const dim3 grid(n_tiles, want < cap ? want : cap);
  if (dtype == kF32) attention_shared_join_kernel<float><<<grid, 256, 0, s>>>(a, static_cast<float*>(out), held);
  else attention_shared_join_kernel<bf16_t><<<grid, 256, 0, s>>>(a, static_cast<bf16_t*>(out), held);
  return check_launch("sp_attention_shared (join)");
}
