// Drafted tokens tested against the target's probabilities with given uniform numbers, and the next token drawn.
//
// Sequence s has rows start .. start + len - 1: token[start] is its last sure token, token[start + 1 + j] its draft j, and row start + j of
// the logits is what the target says of draft j (the last row: of the token after all drafts).  With p = softmax(logits / temperature) and q
// = softmax(draft logits / temperature) of the row that the draft was drawn from (without one: q is 1 at the draft), draft j holds while
// u[start + j] q(draft) < p(draft).  At the first that does not, the next token is drawn from max(p - q, 0), after the last from p: the
// lowest index whose running sum exceeds u[start + len - 1] times the whole sum.  That leaves every token distributed as the target has it.
// Temperature 0: draft j holds while it is the lowest index of the row's maximum, which is the next token.
//
// The answers are whole numbers, and a running sum over 150,000 tokens passes as many borders: exponentials and sums are float64, whose
// errors here (2e-10 of a weight that is compared or drawn from, 1e-9 of a row's sum) move an answer once in millions of draws; float32
// sums would once in a thousand.  Reading the rows' logits bounds the whole.  So that it takes longer than weighing them, sums use a
// table and a float32 polynomial, single weights a float64 polynomial of degree 8 (the library's exponential took 184 us of 646 rows
// of 152,064, the float64 polynomial 110, this 70 to 76).
//
// Four launches: maximum and sum of every row by chunks, so that few rows fill the chip as many do; a block per sequence, a wave a row,
// joins them and finds the deciding row; a block per chunk and sequence sums what is left there; a block per sequence finds chunk and token.
// For few sequences the third launch does the second's work too (kDecidingBlocks).
// 64 sequences of up to 7 drafts over 152,064 tokens of float32, 354 MB: 70, 7.7, 20.8 and 11.3 us, 3.1 TB/s over all and 5.0 in the first.
// (The third and fourth in one, a sequence's last block drawing: 148 us where the two take 32, for the fences by which its blocks hand over
// their sums drop an XCD's L2.)
#include "common.h"
#include "sprout_hip.h"

namespace sprout {

namespace {

constexpr int kVerifyChunk = 4096;      // logits of a block: 16 a thread

struct ChunkStat { double sum; float top; int32_t best; };      // sum of exp((l - top) / temperature), or (greedy) the lowest index of top; best -1: NaN or +infinity
struct RowStat { double sum; float top; int32_t best; };
struct Decision { double p_scale, q_scale, degree, u; float p_top, q_top; int32_t row, draft_row, draft, kind; };      // kind: 0 from p, 1 from what is left, 2 settled; u: the last uniform number

struct VerifyArgs {
  const void *logits, *draft_logits;
  const int32_t *tokens, *starts, *lens, *draft_rows;
  const float *uniform, *temperature;
  int32_t *accepted, *next;
  ChunkStat *stats;          // [2][rows][chunks]: the target's, then the drafter's by the draft's place among the tokens
  double* left;              // [sequences][chunks]
  Decision* decisions;       // [sequences]
  int rows, drafted, sequences, vocab, chunks;
};

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ void better(float& v, int& i, float ov, int oi) {
  if (ov > v || (ov == v && oi < i)) { v = ov; i = oi; }
}
// 2^y for y <= 0, 0 where that has no float64 (a token that is not allowed weighs nothing): 2^n times the Taylor polynomial of 2^f, whose
// coefficients are ln(2)^k / k!, of degree 8 (2e-10 of the value).  y + 1.5 * 2^52 leaves n in the low word of the sum.
__device__ __forceinline__ double two_to(double y) {
  y = fmax(y, -1100.0);
  const double shifted = y + 6755399441055744.0, f = y - (shifted - 6755399441055744.0);
  const int n = int(__double_as_longlong(shifted));
  double p = 1.3215486790144310e-06;
  p = fma(p, f, 1.5252733804059840e-05);
  p = fma(p, f, 1.5403530393381610e-04);
  p = fma(p, f, 1.3333558146428443e-03);
  p = fma(p, f, 9.6181291076284772e-03);
  p = fma(p, f, 5.5504108664821580e-02);
  p = fma(p, f, 2.4022650695910072e-01);
  p = fma(p, f, 6.9314718055994531e-01);
  p = fma(p, f, 1.0);
  return ldexp(p, n);
}
// The same for the sums over whole rows, to 1e-9 of the value, with six float64 instructions (they take twice a float32's time) for sixteen:
// y with 32 bits behind the point is the low word of y + 1.5 * 2^20 and n the bits above it; 2^f is a table's 2^(k / 64) times 1 + a
// cubic in what is left, at most 0.011, which float32 holds to 1e-9.  2^-1000 below that, which no sum notices.
__device__ __forceinline__ double table_power(const double* table, double diff, double degree) {
  const long long bits = __double_as_longlong(fmax(diff * degree, -1000.0) + 1572864.0);
  const uint32_t low = uint32_t(bits);
  const float r = float(low & 0x03ffffffu) * 0x1p-32f;
  const double t = table[low >> 26];
  const float q = r * fmaf(r, fmaf(r, 5.5504109e-02f, 2.4022651e-01f), 6.9314718e-01f);
  const long long power = __double_as_longlong(fma(t, double(q), t));
  return __longlong_as_double((long long)(uint32_t(power >> 32) + (uint32_t(bits >> 32) << 20)) << 32 | uint32_t(power));
}
// Temperatures are handled as `degree` = log2(e) / temperature: a logit weighs 2^((l - top) degree).  (The difference first: a product of
// the largest logits rounds by more than any difference.)
__device__ __forceinline__ double degree_of(float temperature) { return 1.4426950408889634 / double(temperature); }
__device__ __forceinline__ double weight(float l, double top, double degree) { return two_to((double(l) - top) * degree); }
__device__ __forceinline__ bool rows_there(const VerifyArgs& a, int start, int len) { return len > 0 && start >= 0 && start <= a.rows - len; }
__device__ __forceinline__ float temperature_of(const VerifyArgs& a, int s) { return a.temperature ? a.temperature[s] : 0.f; }

// Sixteen logits of a chunk to a thread: groups of four, 1,024 apart (VEC), or single ones 256 apart.  What lies behind the row is -infinity.
template <typename T, bool VEC> __device__ __forceinline__ int logit_index(int chunk, int j) {
  return chunk * kVerifyChunk + (VEC ? 4 * int(threadIdx.x) + 1024 * (j / 4) + j % 4 : int(threadIdx.x) + 256 * j);
}
__device__ __forceinline__ void load_four(const float* row, int i, int vocab, float* v) {      // (vocab is whole fours)
  const float4 x = i < vocab ? *reinterpret_cast<const float4*>(row + i) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
  v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
}
__device__ __forceinline__ void load_four(const bf16_t* row, int i, int vocab, float* v) {
  const uint2 x = i < vocab ? *reinterpret_cast<const uint2*>(row + i) : make_uint2(0xff80ff80u, 0xff80ff80u);
  v[0] = __uint_as_float(x.x << 16); v[1] = __uint_as_float(x.x & 0xffff0000u);
  v[2] = __uint_as_float(x.y << 16); v[3] = __uint_as_float(x.y & 0xffff0000u);
}
template <typename T, bool VEC> __device__ __forceinline__ void load_logits(const T* row, int chunk, int vocab, float (&v)[16]) {
#pragma unroll
  for (int j = 0; j < 16; j += VEC ? 4 : 1) {
    const int i = logit_index<T, VEC>(chunk, j);
    if (VEC) load_four(row, i, vocab, v + j);
    else v[j] = i < vocab ? to_float(row[i]) : -INFINITY;
  }
}

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void verify_stats_kernel(VerifyArgs a) {
  __shared__ double s_powers[64];
  __shared__ float s_top[4];
  __shared__ int s_best, s_seq;
  __shared__ double s_sum[4];
  const int chunk = blockIdx.x, place = int(blockIdx.y) >= a.rows ? blockIdx.y - a.rows : blockIdx.y;
  const bool drafter = int(blockIdx.y) >= a.rows;
  int row = place;
  if (drafter) {
    row = a.draft_rows[place];
    if (row < 0 || row >= a.drafted) return;
  }
  // the row is asked for before it is known whose it is
  float v[16];
  load_logits<T, VEC>(static_cast<const T*>(drafter ? a.draft_logits : a.logits) + size_t(row) * a.vocab, chunk, a.vocab, v);
  if (threadIdx.x < 64) s_powers[threadIdx.x] = two_to(double(threadIdx.x) / 64.0 - 1.0) * 2.0;
  if (threadIdx.x == 0) { s_seq = -1; s_best = 0x7fffffff; }
  __syncthreads();
  for (int s = threadIdx.x; s < a.sequences; s += 256) {
    const int start = a.starts[s], len = a.lens[s];
    if (rows_there(a, start, len) && place >= start + (drafter ? 1 : 0) && place - start < len) s_seq = s;
  }
  __syncthreads();
  const int seq = s_seq;
  if (seq < 0) return;
  const float temp = temperature_of(a, seq);
  if (drafter && !(temp > 0.f)) return;
  const bool greedy = !(temp > 0.f);
  // the maximum that is NaN where a number is: NaN and +infinity make a row that is not taken
  float top = v[0];
#pragma unroll
  for (int j = 1; j < 16; ++j) top = __builtin_elementwise_maximum(top, v[j]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = __builtin_elementwise_maximum(top, __shfl_xor(top, o, 64));
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) s_top[wave] = top;
  __syncthreads();
  for (int w = 0; w < 4; ++w) top = __builtin_elementwise_maximum(top, s_top[w]);
  const bool good = top < INFINITY;
  int best = 0x7fffffff;
  double sum = 0.0;
  if (greedy) {
#pragma unroll
    for (int j = 15; j >= 0; --j) {
      const int i = logit_index<T, VEC>(chunk, j);
      if (i < a.vocab && v[j] == top) best = min(best, i);
    }
    if (best != 0x7fffffff) atomicMin(&s_best, best);
  } else if (good && top > -INFINITY) {
    const double degree = degree_of(temp), from = double(top);
    double sums[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
    for (int j = 0; j < 16; ++j) sums[j % 4] += table_power(s_powers, double(v[j]) - from, degree);
    sum = wave_sum64((sums[0] + sums[1]) + (sums[2] + sums[3]));
    if ((threadIdx.x & 63) == 0) s_sum[wave] = sum;
  }
  __syncthreads();
  if (threadIdx.x == 0)
    a.stats[(size_t(blockIdx.y)) * a.chunks + chunk] = {greedy || !(top > -INFINITY) || !good ? 0.0 : s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3], top,
                                                        !good ? -1 : greedy ? s_best : 0};
}

// A wave: the statistics of one row from its chunks'.  best -1: NaN, +infinity, or nothing but -infinity.
__device__ __forceinline__ RowStat row_stat(const ChunkStat* stats, int chunks, double degree) {
  const int lane = threadIdx.x & 63;
  float top = -INFINITY;
  int best = 0x7fffffff, bad = 0;
  const ChunkStat first = lane < chunks ? stats[lane] : ChunkStat{0.0, -INFINITY, 0x7fffffff};
  for (int c = lane; c < chunks; c += 64) {
    const ChunkStat st = c == lane ? first : stats[c];
    if (st.best < 0) bad = 1;
    better(top, best, st.top, st.best);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float ov = __shfl_xor(top, o, 64);
    const int oi = __shfl_xor(best, o, 64);
    better(top, best, ov, oi);
    bad |= __shfl_xor(bad, o, 64);
  }
  double sum = 0.0;
  for (int c = lane; c < chunks; c += 64) {
    const ChunkStat st = c == lane ? first : stats[c];
    if (st.top > -INFINITY) sum += st.sum * weight(st.top, double(top), degree);
  }
  return {wave_sum64(sum), top, bad || !(top > -INFINITY) ? -1 : best};
}

// A sequence's deciding row, into `found` (shared memory; a barrier follows); `say`: this block writes the answers down.  kRows waves take that
// many rows at a time; the last row of a sequence never holds.
template <typename T, int kRows> __device__ __forceinline__ void decide(const VerifyArgs& a, int seq, bool say, Decision& found) {
  __shared__ Decision s_found[kRows];
  __shared__ int s_holds[kRows], s_next[kRows];
  const int wave = threadIdx.x >> 6;
  const int start = a.starts[seq], len = a.lens[seq];
  bool refused = !rows_there(a, start, len);
  for (int s = threadIdx.x; s < a.sequences; s += 64 * kRows) {
    const int other = a.starts[s], n = a.lens[s];
    if (s != seq && !refused && rows_there(a, other, n) && other < start + len && start < other + n) refused = true;
  }
  if (__syncthreads_or(refused)) {      // rows that are not there, or also another sequence's, whose temperature may differ
    if (threadIdx.x == 0) {
      found.kind = 2;
      if (say) { a.accepted[seq] = 0; a.next[seq] = -1; a.decisions[seq].kind = 2; }
    }
    return;
  }
  const float temp = temperature_of(a, seq);
  const bool greedy = !(temp > 0.f);
  const double degree = greedy ? 0.0 : degree_of(temp), last_u = greedy ? 0.0 : double(a.uniform[start + len - 1]);
  for (int first = 0;; first += kRows) {
    const int j = first + wave;
    if (j < len) {
      const int place = start + j;
      const bool tested = j < len - 1;
      const int draft = tested ? a.tokens[place + 1] : -1, from = tested && a.draft_rows && !greedy ? a.draft_rows[place + 1] : -1;
      const bool known = draft >= 0 && draft < a.vocab, drawn = from >= 0 && from < a.drafted;
      // all that the row needs is asked for together
      const float l_p = known ? to_float(static_cast<const T*>(a.logits)[size_t(place) * a.vocab + draft]) : 0.f;
      const float l_q = known && drawn ? to_float(static_cast<const T*>(a.draft_logits)[size_t(from) * a.vocab + draft]) : 0.f;
      const float u = tested && !greedy ? a.uniform[place] : 0.f;
      RowStat q = {1.0, 0.f, -1};
      if (drawn) q = row_stat(a.stats + (size_t(a.rows) + place + 1) * a.chunks, a.chunks, degree);
      const RowStat p = row_stat(a.stats + size_t(place) * a.chunks, a.chunks, degree);
      Decision mine = {1.0 / p.sum, 0.0, degree, last_u, p.top, 0.f, place, -1, -1, tested ? 1 : 0};
      bool holds = false;
      int token = p.best;      // what is next where the row settles that without a draw: the greedy choice, or -1
      if (p.best < 0 || greedy) {
        mine.kind = 2;
        holds = p.best >= 0 && tested && draft == p.best;
      } else if (tested) {
        mine.draft = draft;
        double q_draft = 1.0;
        if (from >= 0) {
          mine.draft_row = from;
          mine.q_scale = 1.0 / q.sum;
          mine.q_top = q.top;
          if (q.best < 0) { mine.kind = 2; token = -1; }
          else q_draft = weight(l_q, double(q.top), degree) * mine.q_scale;
        }
        holds = mine.kind == 1 && known && double(u) * q_draft < weight(l_p, double(p.top), degree) * mine.p_scale;
      }
      if ((threadIdx.x & 63) == 0) { s_found[wave] = mine; s_holds[wave] = holds; s_next[wave] = token; }
    }
    __syncthreads();
    const int n = min(kRows, len - first);
    int stop = 0;
    while (stop < n && s_holds[stop]) ++stop;
    if (stop < n) {      // (the same in every thread)
      if (threadIdx.x == 0) {
        found = s_found[stop];
        if (say) {
          a.accepted[seq] = first + stop;
          a.decisions[seq] = s_found[stop];
          if (s_found[stop].kind == 2) a.next[seq] = s_next[stop];
        }
      }
      return;
    }
    __syncthreads();
  }
}

template <typename T> __global__ __launch_bounds__(512) void verify_decide_kernel(VerifyArgs a) {
  __shared__ Decision found;
  decide<T, 8>(a, blockIdx.x, true, found);
}

// What is left of a token's probability in the deciding row, of logits p and q (drawn: q from the drafter's row).  kind 0: all of it, else
// what p has more than q.
__device__ __forceinline__ double left_of(const Decision& d, bool drawn, double degree, float p, float q, int token) {
  const double mine = weight(p, double(d.p_top), degree) * d.p_scale;
  if (d.kind == 0) return mine;
  const double other = drawn ? weight(q, double(d.q_top), degree) * d.q_scale : token == d.draft ? 1.0 : 0.0;
  return mine > other ? mine - other : 0.0;
}

// What is left in a chunk of the deciding row.  DECIDES: every block of a sequence finds that row itself, with twice the waves.  (Loops that are not
// unrolled over a thread's logits: few blocks run this, and code that is run once costs its own way from memory.)
template <typename T, bool VEC, bool DECIDES>
__global__ __launch_bounds__(DECIDES ? 512 : 256) void verify_left_kernel(VerifyArgs a) {
  constexpr int kThreads = DECIDES ? 512 : 256, kGroups = kVerifyChunk / (4 * kThreads);
  __shared__ double s_sum[kThreads / 64];
  __shared__ Decision s_decision;
  const int chunk = blockIdx.x, seq = blockIdx.y, wave = threadIdx.x >> 6;
  if (DECIDES) {
    decide<T, kThreads / 64>(a, seq, chunk == 0, s_decision);
    __syncthreads();
  }
  const Decision d = DECIDES ? s_decision : a.decisions[seq];
  if (d.kind == 2) return;
  const bool drawn = d.kind == 1 && d.draft_row >= 0;
  const T* row = static_cast<const T*>(a.logits) + size_t(d.row) * a.vocab;
  const T* draft_row = drawn ? static_cast<const T*>(a.draft_logits) + size_t(d.draft_row) * a.vocab : row;
  const double degree = d.degree;
  float p[4], q[4];
  auto first_of = [&](int group) { return chunk * kVerifyChunk + 4 * kThreads * group + (VEC ? 4 : 1) * int(threadIdx.x); };
  auto load = [&](int group) __attribute__((always_inline)) {
    const int i = first_of(group);
    if (VEC) {
      load_four(row, i, a.vocab, p);
      load_four(draft_row, i, a.vocab, q);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        p[j] = i + kThreads * j < a.vocab ? to_float(row[i + kThreads * j]) : -INFINITY;
        q[j] = i + kThreads * j < a.vocab ? to_float(draft_row[i + kThreads * j]) : -INFINITY;
      }
    }
  };
  double sum = 0.0;
  load(0);
#pragma unroll 1
  for (int group = 0; group < kGroups; ++group) {
    const float p_now[4] = {p[0], p[1], p[2], p[3]}, q_now[4] = {q[0], q[1], q[2], q[3]};
    if (group + 1 < kGroups) load(group + 1);
#pragma unroll
    for (int j = 0; j < 4; ++j) sum += left_of(d, drawn, degree, p_now[j], q_now[j], first_of(group) + (VEC ? j : kThreads * j));
  }
  sum = wave_sum64(sum);
  if ((threadIdx.x & 63) == 0) s_sum[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double all = 0.0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) all += s_sum[w];
    a.left[size_t(seq) * a.chunks + chunk] = all;
  }
}

constexpr int kDrawThreads = kVerifyChunk / 4;
// The sum of v over the threads before this one; `total`: over all.
__device__ __forceinline__ double sum_before(double v, double* scratch, double& total) {
  constexpr int WAVES = kDrawThreads / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double running = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double add = __shfl_up(running, o, 64);
    if (lane >= o) running += add;
  }
  __syncthreads();      // what lay in `scratch` has been used
  if (lane == 63) scratch[wave] = running;
  __syncthreads();
  double before = __shfl_up(running, 1, 64), waves = lane < WAVES ? scratch[lane] : 0.0;
  if (lane == 0) before = 0.0;
#pragma unroll
  for (int o = 1; o < WAVES; o <<= 1) {
    const double add = __shfl_up(waves, o, 64);
    if (lane >= o) waves += add;
  }
  total = __shfl(waves, WAVES - 1, 64);
  const double of_waves = __shfl(waves, wave - 1 & 63, 64);
  return wave ? before + of_waves : before;
}

// A block per sequence, a thread a chunk and then four tokens of the chunk that the limit lies in.
template <typename T, bool VEC>
__global__ __launch_bounds__(kDrawThreads) void verify_draw_kernel(VerifyArgs a) {
  __shared__ double s_scratch[kDrawThreads / 64], s_before;
  __shared__ int s_chunk, s_token, s_last;
  const int seq = blockIdx.x, t = threadIdx.x;
  Decision d = a.decisions[seq];
  if (d.kind == 2) return;
  // ---- the chunk: a thread has one, or a run of them (a vocabulary of more than four million)
  const int per = (a.chunks + kDrawThreads - 1) / kDrawThreads, from = min(t * per, a.chunks), to = min(from + per, a.chunks);
  double mine = 0.0, total = 0.0, before = 0.0, found_before = 0.0, last_before = 0.0;
  int found = 0x7fffffff, last = -1;
  if (t == 0) { s_chunk = 0x7fffffff; s_last = -1; s_token = 0x7fffffff; }
  const double* left = a.left + size_t(seq) * a.chunks;
  const ChunkStat* stats = a.stats + size_t(d.row) * a.chunks;
#pragma unroll 1
  for (int turn = 0; turn < 2; ++turn) {
    auto mass = [&](int c) {      // the second turn: nothing is left of p - q, and the next token comes from p
      return turn == 0 ? left[c] : stats[c].top > -INFINITY ? stats[c].sum * weight(stats[c].top, double(d.p_top), d.degree) * d.p_scale : 0.0;
    };
    mine = 0.0;
#pragma unroll 1
    for (int c = from; c < to; ++c) mine += mass(c);
    before = sum_before(mine, s_scratch, total);
    double running = before;
#pragma unroll 1
    for (int c = from; c < to; ++c) {
      const double m = per == 1 ? mine : mass(c);
      if (m > 0.0) {
        last = c;
        last_before = running;
        if (running + m > d.u * total && found == 0x7fffffff) { found = c; found_before = running; }
      }
      running += m;
    }
    if (total > 0.0 || d.kind == 0) break;
    d.kind = 0;      // (a draft that neither side allows, under equal rows)
  }
  const double limit = d.u * total;
  if (found != 0x7fffffff) atomicMin(&s_chunk, found);
  __syncthreads();
  int chunk = s_chunk;
  if (chunk == 0x7fffffff) {      // a limit that rounding has put at the very end: the last chunk of any weight
    if (last >= 0) atomicMax(&s_last, last);
    __syncthreads();
    chunk = s_last;
  }
  if (chunk < 0) {
    if (t == 0) a.next[seq] = -1;
    return;
  }
  if (chunk >= from && chunk < to) s_before = found == chunk ? found_before : last_before;
  // ---- the token
  const bool drawn = d.kind == 1 && d.draft_row >= 0;
  const T* row = static_cast<const T*>(a.logits) + size_t(d.row) * a.vocab;
  const T* draft_row = drawn ? static_cast<const T*>(a.draft_logits) + size_t(d.draft_row) * a.vocab : row;
  const int begin = chunk * kVerifyChunk + 4 * t;
  float p[4], q[4];
  if (VEC) {
    load_four(row, begin, a.vocab, p);
    load_four(draft_row, begin, a.vocab, q);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      p[j] = begin + j < a.vocab ? to_float(row[begin + j]) : -INFINITY;
      q[j] = begin + j < a.vocab ? to_float(draft_row[begin + j]) : -INFINITY;
    }
  }
  double w[4], in_chunk;
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = left_of(d, drawn, d.degree, p[j], q[j], begin + j);
  double running = sum_before(((w[0] + w[1]) + w[2]) + w[3], s_scratch, in_chunk) + s_before;
  found = 0x7fffffff;
  last = -1;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    running += w[j];
    if (w[j] > 0.0) {
      last = begin + j;
      if (running > limit && found == 0x7fffffff) found = begin + j;
    }
  }
  if (found != 0x7fffffff) atomicMin(&s_token, found);
  __syncthreads();
  if (s_token == 0x7fffffff) {      // likewise within the chunk
    if (t == 0) s_last = -1;
    __syncthreads();
    if (last >= 0) atomicMax(&s_last, last);
    __syncthreads();
    if (t == 0) a.next[seq] = s_last;
  } else if (t == 0) {
    a.next[seq] = s_token;
  }
}

int chunks_of(int vocab) { return (vocab + kVerifyChunk - 1) / kVerifyChunk; }
size_t verify_bytes(int rows, int sequences, int vocab) {
  const size_t c = chunks_of(vocab);
  return 2 * size_t(rows) * c * sizeof(ChunkStat) + size_t(sequences) * c * sizeof(double) + size_t(sequences) * sizeof(Decision);
}

// Up to so many blocks of what is left decide by themselves: one launch less, but the same work in every block of a sequence (rows of 151,936: 1,
// 4, 9, 20 sequences 22.1, 24.3, 32.4, 41.5 us and 24.3, 26.8, 34.6, 43.4 with a launch of its own; 27, 40, 64 sequences 54.9, 70.9, 124 and 52.5, 65.6, 110).
constexpr int kDecidingBlocks = 768;

template <typename T, bool VEC> int launch_verify(hipStream_t s, const VerifyArgs& a) {
  verify_stats_kernel<T, VEC><<<dim3(a.chunks, a.rows * (a.draft_logits ? 2 : 1)), 256, 0, s>>>(a);
  const bool few = a.temperature && int64_t(a.chunks) * a.sequences <= kDecidingBlocks;
  if (!few) verify_decide_kernel<T><<<a.sequences, 512, 0, s>>>(a);
  if (a.temperature) {
    if (few) verify_left_kernel<T, VEC, true><<<dim3(a.chunks, a.sequences), 512, 0, s>>>(a);
    else verify_left_kernel<T, VEC, false><<<dim3(a.chunks, a.sequences), 256, 0, s>>>(a);
    verify_draw_kernel<T, VEC><<<a.sequences, kDrawThreads, 0, s>>>(a);
  }
  return check_launch("sp_verify_drafts");
}

}  // namespace

}  // namespace sprout

using namespace sprout;

extern "C" int64_t sp_verify_workspace_floats(int rows, int sequences, int vocab) {
  return rows <= 0 || sequences <= 0 || vocab <= 0 ? 0 : int64_t(verify_bytes(rows, sequences, vocab) / 4);
}

extern "C" int sp_verify_drafts(void* stream, int dtype, const void* logits, int rows, int vocab, const int32_t* tokens, const int32_t* starts,
                                const int32_t* lens, int sequences, const float* uniform, const float* temperature, const void* draft_logits,
                                int drafted, const int32_t* draft_rows, int32_t* accepted, int32_t* next, void* workspace,
                                int64_t workspace_floats) {
  SP_REQUIRE(dtype == kF32 || dtype == kBF16, "sp_verify_drafts: unsupported dtype %d", dtype);
  SP_REQUIRE(rows >= 0 && sequences >= 0 && vocab > 0 && vocab <= 1 << 30 && drafted >= 0, "sp_verify_drafts: bad sizes rows=%d sequences=%d vocab=%d drafted=%d", rows, sequences, vocab, drafted);
  if (sequences == 0) return 0;
  SP_REQUIRE(rows > 0 && rows <= 32767, "sp_verify_drafts: %d rows are outside 1..32767", rows);
  SP_REQUIRE(sequences <= 65535, "sp_verify_drafts: %d sequences are more than 65535", sequences);
  SP_REQUIRE(logits && tokens && starts && lens && accepted && next && (uniform || !temperature), "sp_verify_drafts: null argument");
  SP_REQUIRE(!draft_logits == !draft_rows || (draft_rows && drafted == 0), "sp_verify_drafts: draft logits and the rows of the drafts go together");
  const int64_t need = sp_verify_workspace_floats(rows, sequences, vocab);
  SP_REQUIRE(workspace && workspace_floats >= need && reinterpret_cast<uintptr_t>(workspace) % 8 == 0,
             "sp_verify_drafts: workspace of %lld floats, %lld needed at a multiple of 8 bytes", (long long)workspace_floats, (long long)need);
  VerifyArgs a;
  a.logits = logits; a.draft_logits = temperature && drafted ? draft_logits : nullptr;
  a.tokens = tokens; a.starts = starts; a.lens = lens; a.draft_rows = draft_rows;
  a.uniform = uniform; a.temperature = temperature; a.accepted = accepted; a.next = next;
  a.rows = rows; a.drafted = drafted; a.sequences = sequences; a.vocab = vocab; a.chunks = chunks_of(vocab);
  a.stats = static_cast<ChunkStat*>(workspace);
  a.left = reinterpret_cast<double*>(a.stats + 2 * size_t(rows) * a.chunks);
  a.decisions = reinterpret_cast<Decision*>(a.left + size_t(sequences) * a.chunks);
  // rows of whole groups of four that start where four lie in one load
  const uintptr_t starts_at = reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(a.draft_logits);
  const bool vec = vocab % 4 == 0 && starts_at % (dtype == kF32 ? 16 : 8) == 0;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == kF32) return vec ? launch_verify<float, true>(s, a) : launch_verify<float, false>(s, a);
  return vec ? launch_verify<bf16_t, true>(s, a) : launch_verify<bf16_t, false>(s, a);
}
