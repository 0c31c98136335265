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
// vector rate equals float32's here, so that the sum's order moves an answer about once in 10^11 draws (float32: once in a thousand).
//
// Three launches: maximum and sum of every row by chunks, so that few rows fill the chip as many do; then a block per chunk and sequence
// joins the chunks' statistics, finds the deciding row and sums its chunk of what is left; then a block per sequence finds chunk and token.
#include "common.h"
#include "sprout_hip.h"

namespace sprout {

namespace {

constexpr int kVerifyChunk = 4096;      // logits of a block: 16 a thread

struct ChunkStat { double sum; float top; int32_t best; };                   // sum of exp((l - top) / temperature); best: index of top, -1: no good row
struct RowStat { double sum; float top; int32_t best; };
struct Decision { double p_scale, q_scale; float p_top, q_top; int32_t row, draft_row, draft, kind; };   // kind: 0 from p, 1 from what is left, 2 settled

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
__device__ __forceinline__ double weight(float l, float top, double per_degree) {
  return l == -INFINITY ? 0.0 : exp((double(l) - double(top)) * per_degree);
}
__device__ __forceinline__ float temperature_of(const VerifyArgs& a, int s) { return a.temperature ? a.temperature[s] : 0.f; }

template <typename T>
__global__ __launch_bounds__(256) void verify_stats_kernel(VerifyArgs a) {
  __shared__ float s_top[4];
  __shared__ int s_best[4], s_seq, s_bad;
  __shared__ double s_sum[4];
  const int chunk = blockIdx.x, place = blockIdx.y % a.rows;
  const bool drafter = int(blockIdx.y) >= a.rows;
  if (threadIdx.x == 0) { s_seq = -1; s_bad = 0; }
  __syncthreads();
  for (int s = threadIdx.x; s < a.sequences; s += 256) {
    const int at = place - a.starts[s];
    if (at >= (drafter ? 1 : 0) && at < a.lens[s]) s_seq = s;
  }
  __syncthreads();
  const int seq = s_seq;
  if (seq < 0) return;
  const float temp = temperature_of(a, seq);
  int row = place;
  if (drafter) {
    row = a.draft_rows[place];
    if (!(temp > 0.f) || row < 0 || row >= a.drafted) return;
  }
  const T* src = static_cast<const T*>(drafter ? a.draft_logits : a.logits) + size_t(row) * a.vocab;
  const int begin = chunk * kVerifyChunk;
  float v[16], top = -INFINITY;
  int best = 0x7fffffff;
  bool bad = false;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const int i = begin + threadIdx.x + 256 * j;
    v[j] = i < a.vocab ? to_float(src[i]) : -INFINITY;
    bad |= !(v[j] < INFINITY);      // NaN or +infinity; a token whose logit is -infinity has probability 0
    if (i < a.vocab) better(top, best, v[j], i);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) better(top, best, __shfl_xor(top, o, 64), __shfl_xor(best, o, 64));
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) { s_top[wave] = top; s_best[wave] = best; }
  if (bad) s_bad = 1;
  __syncthreads();
  for (int w = 0; w < 4; ++w) better(top, best, s_top[w], s_best[w]);
  double sum = 0.0;
  if (temp > 0.f && top > -INFINITY) {
    const double per_degree = 1.0 / double(temp);
#pragma unroll
    for (int j = 0; j < 16; ++j) sum += weight(v[j], top, per_degree);
  }
  sum = wave_sum64(sum);
  if ((threadIdx.x & 63) == 0) s_sum[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0)
    a.stats[(size_t(blockIdx.y)) * a.chunks + chunk] = {s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3], top, s_bad ? -1 : best};
}

// A wave: the statistics of one row from its chunks'.  best -1: NaN, +infinity, or nothing but -infinity.
__device__ __forceinline__ RowStat row_stat(const ChunkStat* stats, int chunks, double per_degree) {
  const int lane = threadIdx.x & 63;
  float top = -INFINITY;
  int best = 0x7fffffff, bad = 0;
  for (int c = lane; c < chunks; c += 64) {
    const ChunkStat st = stats[c];
    if (st.best < 0) bad = 1;
    better(top, best, st.top, st.best);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    better(top, best, __shfl_xor(top, o, 64), __shfl_xor(best, o, 64));
    bad |= __shfl_xor(bad, o, 64);
  }
  double sum = 0.0;
  for (int c = lane; c < chunks; c += 64) sum += stats[c].sum * weight(stats[c].top, top, per_degree);
  return {wave_sum64(sum), top, bad || !(top > -INFINITY) ? -1 : best};
}

// What is left of token i's probability in the deciding row.
template <typename T> __device__ __forceinline__ double left_of(const Decision& d, const T* row, const T* draft_row, int i, double per_degree) {
  const double p = weight(to_float(row[i]), d.p_top, per_degree) * d.p_scale;
  if (d.kind == 0) return p;
  const double q = draft_row ? weight(to_float(draft_row[i]), d.q_top, per_degree) * d.q_scale : i == d.draft ? 1.0 : 0.0;
  return p > q ? p - q : 0.0;
}

template <typename T>
__global__ __launch_bounds__(256) void verify_decide_kernel(VerifyArgs a) {
  __shared__ Decision s_found[4];
  __shared__ int s_holds[4], s_next[4];
  __shared__ double s_sum[4];
  const int chunk = blockIdx.x, seq = blockIdx.y, wave = threadIdx.x >> 6;
  const int start = a.starts[seq], len = a.lens[seq];
  if (len <= 0 || start < 0 || start > a.rows - len) {      // rows that are not there
    if (chunk == 0 && threadIdx.x == 0) { a.accepted[seq] = 0; a.next[seq] = -1; a.decisions[seq].kind = 2; }
    return;
  }
  const float temp = temperature_of(a, seq);
  const bool greedy = !(temp > 0.f);
  const double per_degree = greedy ? 0.0 : 1.0 / double(temp);
  int accepted = -1;
  Decision d;
  int next = -1;
  for (int first = 0; accepted < 0; first += 4) {      // four drafts at a time; the last row of a sequence never holds
    const int j = first + wave;
    if (j < len) {
      const int place = start + j;
      const RowStat p = row_stat(a.stats + size_t(place) * a.chunks, a.chunks, per_degree);
      Decision mine = {1.0 / p.sum, 0.0, p.top, 0.f, place, -1, -1, 0};
      bool holds = false;
      int token = p.best;      // what is next where the row settles that without a draw: the greedy choice, or -1
      if (p.best < 0) {
        mine.kind = 2;
      } else if (greedy) {
        mine.kind = 2;
        holds = j < len - 1 && a.tokens[place + 1] == p.best;
      } else if (j < len - 1) {
        const int draft = a.tokens[place + 1];
        const int from = a.draft_rows ? a.draft_rows[place + 1] : -1;
        const bool known = draft >= 0 && draft < a.vocab;
        double q_draft = 1.0;
        mine.kind = 1;
        mine.draft = draft;
        if (from >= 0) {
          mine.draft_row = from;
          const RowStat q = from < a.drafted ? row_stat(a.stats + (size_t(a.rows) + place + 1) * a.chunks, a.chunks, per_degree)
                                             : RowStat{1.0, 0.f, -1};
          if (q.best < 0) { mine.kind = 2; token = -1; }
          else {
            mine.q_scale = 1.0 / q.sum;
            mine.q_top = q.top;
            q_draft = known ? weight(to_float(static_cast<const T*>(a.draft_logits)[size_t(from) * a.vocab + draft]), q.top, per_degree) * mine.q_scale : 0.0;
          }
        }
        if (mine.kind == 1 && known) {
          const double p_draft = weight(to_float(static_cast<const T*>(a.logits)[size_t(place) * a.vocab + draft]), p.top, per_degree) * mine.p_scale;
          holds = double(a.uniform[place]) * q_draft < p_draft;
        }
      }
      if ((threadIdx.x & 63) == 0) { s_found[wave] = mine; s_holds[wave] = holds; s_next[wave] = token; }
    }
    __syncthreads();
    for (int w = 0; w < 4 && accepted < 0; ++w)
      if (first + w < len && !s_holds[w]) { accepted = first + w; d = s_found[w]; next = s_next[w]; }
    __syncthreads();
  }
  if (chunk == 0 && threadIdx.x == 0) {
    a.accepted[seq] = accepted;
    a.decisions[seq] = d;
    if (d.kind == 2) a.next[seq] = next;
  }
  if (d.kind == 2) return;
  const T* row = static_cast<const T*>(a.logits) + size_t(d.row) * a.vocab;
  const T* draft_row = d.draft_row >= 0 ? static_cast<const T*>(a.draft_logits) + size_t(d.draft_row) * a.vocab : nullptr;
  double sum = 0.0;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const int i = chunk * kVerifyChunk + threadIdx.x + 256 * j;
    if (i < a.vocab) sum += left_of(d, row, draft_row, i, per_degree);
  }
  sum = wave_sum64(sum);
  if ((threadIdx.x & 63) == 0) s_sum[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) a.left[size_t(seq) * a.chunks + chunk] = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
}

template <typename T>
__global__ __launch_bounds__(256) void verify_draw_kernel(VerifyArgs a) {
  __shared__ double s_scan[256], s_before, s_limit;
  __shared__ int s_chunk, s_token, s_last;
  const int seq = blockIdx.x;
  Decision d = a.decisions[seq];
  if (d.kind == 2) return;
  const double per_degree = 1.0 / double(temperature_of(a, seq));
  const double u = double(a.uniform[a.starts[seq] + a.lens[seq] - 1]);
  const ChunkStat* stats = a.stats + size_t(d.row) * a.chunks;
  if (threadIdx.x == 0) {
    double total = 0.0;
    for (int c = 0; c < a.chunks; ++c) total += a.left[size_t(seq) * a.chunks + c];
    // nothing is left of p - q (a draft that neither side allows, under equal rows): the next token comes from p
    const bool from_p = d.kind == 1 && !(total > 0.0);
    auto mass = [&](int c) { return from_p ? stats[c].sum * weight(stats[c].top, d.p_top, per_degree) * d.p_scale : a.left[size_t(seq) * a.chunks + c]; };
    if (from_p) {
      total = 0.0;
      for (int c = 0; c < a.chunks; ++c) total += mass(c);
    }
    const double limit = u * total;
    double before = 0.0, running = 0.0;
    int chunk = -1;
    for (int c = 0; c < a.chunks; ++c) {
      const double m = mass(c);
      if (m > 0.0) {
        chunk = c;
        before = running;
        running += m;
        if (running > limit) break;
      }
    }
    s_chunk = chunk; s_before = before; s_limit = limit;
    s_token = from_p ? -2 : 0x7fffffff;
    s_last = -1;
  }
  __syncthreads();
  if (s_token == -2) d.kind = 0;
  __syncthreads();
  if (threadIdx.x == 0) s_token = 0x7fffffff;
  const T* row = static_cast<const T*>(a.logits) + size_t(d.row) * a.vocab;
  const T* draft_row = d.kind == 1 && d.draft_row >= 0 ? static_cast<const T*>(a.draft_logits) + size_t(d.draft_row) * a.vocab : nullptr;
  // sixteen tokens in a row to a thread
  double w[16], sum = 0.0;
  const int begin = s_chunk * kVerifyChunk + 16 * threadIdx.x;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    w[j] = begin + j < a.vocab ? left_of(d, row, draft_row, begin + j, per_degree) : 0.0;
    sum += w[j];
  }
  s_scan[threadIdx.x] = sum;
  __syncthreads();
  for (int o = 1; o < 256; o <<= 1) {
    const double add = int(threadIdx.x) >= o ? s_scan[threadIdx.x - o] : 0.0;
    __syncthreads();
    s_scan[threadIdx.x] += add;
    __syncthreads();
  }
  double running = s_before + (threadIdx.x ? s_scan[threadIdx.x - 1] : 0.0);
  int found = 0x7fffffff, last = -1;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    running += w[j];
    if (w[j] > 0.0) {
      last = begin + j;
      if (running > s_limit && found == 0x7fffffff) found = begin + j;
    }
  }
  if (found != 0x7fffffff) atomicMin(&s_token, found);
  if (last >= 0) atomicMax(&s_last, last);
  __syncthreads();
  // (a limit that rounding has put at the chunk's very end: its last token of any weight)
  if (threadIdx.x == 0) a.next[seq] = s_token != 0x7fffffff ? s_token : s_last;
}

int chunks_of(int vocab) { return (vocab + kVerifyChunk - 1) / kVerifyChunk; }
size_t verify_bytes(int rows, int sequences, int vocab) {
  const size_t c = chunks_of(vocab);
  return 2 * size_t(rows) * c * sizeof(ChunkStat) + size_t(sequences) * c * sizeof(double) + size_t(sequences) * sizeof(Decision);
}

template <typename T> int launch_verify(hipStream_t s, const VerifyArgs& a) {
  verify_stats_kernel<T><<<dim3(a.chunks, a.rows * (a.draft_logits ? 2 : 1)), 256, 0, s>>>(a);
  verify_decide_kernel<T><<<dim3(a.chunks, a.sequences), 256, 0, s>>>(a);
  if (a.temperature) verify_draw_kernel<T><<<a.sequences, 256, 0, s>>>(a);
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
  SP_REQUIRE(rows >= 0 && sequences >= 0 && vocab > 0 && drafted >= 0, "sp_verify_drafts: bad sizes rows=%d sequences=%d vocab=%d drafted=%d", rows, sequences, vocab, drafted);
  if (sequences == 0) return 0;
  SP_REQUIRE(rows > 0 && rows <= 32767, "sp_verify_drafts: %d rows are outside 1..32767", rows);
  SP_REQUIRE(sequences <= 65535, "sp_verify_drafts: %d sequences are more than 65535", sequences);
  SP_REQUIRE(logits && tokens && starts && lens && accepted && next && (uniform || !temperature), "sp_verify_drafts: null argument");
  SP_REQUIRE(!draft_logits == !draft_rows, "sp_verify_drafts: draft logits and the rows of the drafts go together");
  const int64_t need = sp_verify_workspace_floats(rows, sequences, vocab);
  SP_REQUIRE(workspace && workspace_floats >= need && reinterpret_cast<uintptr_t>(workspace) % 8 == 0,
             "sp_verify_drafts: workspace of %lld floats, %lld needed at a multiple of 8 bytes", (long long)workspace_floats, (long long)need);
  VerifyArgs a;
  a.logits = logits; a.draft_logits = temperature && drafted ? draft_logits : nullptr;
  a.tokens = tokens; a.starts = starts; a.lens = lens; a.draft_rows = draft_logits ? draft_rows : nullptr;
  a.uniform = uniform; a.temperature = temperature; a.accepted = accepted; a.next = next;
  a.rows = rows; a.drafted = drafted; a.sequences = sequences; a.vocab = vocab; a.chunks = chunks_of(vocab);
  a.stats = static_cast<ChunkStat*>(workspace);
  a.left = reinterpret_cast<double*>(a.stats + 2 * size_t(rows) * a.chunks);
  a.decisions = reinterpret_cast<Decision*>(a.left + size_t(sequences) * a.chunks);
  return dtype == kF32 ? launch_verify<float>((hipStream_t)stream, a) : launch_verify<bf16_t>((hipStream_t)stream, a);
}
