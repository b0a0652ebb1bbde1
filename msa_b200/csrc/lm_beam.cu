// Beam search: the choice of the next beams from the logits, and the reordering of the sequence states that follows from it.
//
// Choice.  A candidate (beam b, token t) has the score  s_b + (x_bt - lse_b),  lse_b = log sum_t exp x_bt.  Within a row the order is
// that of the logits, so one pass over a row yields both its sum and its k best logits; the second kernel joins a question's rows in
// 64 bits.  Bound by the one read of the logits.
//
// Reordering.  New beam j continues beam parent[j].  Its first child keeps a beam's slot, the others take slots that nobody
// continues: sources and destinations never meet, and no second buffer is needed.  Bound by the copied bytes, read and written once.
#include "lm_common.cuh"

namespace msa {

constexpr int kBeamMax = 32;             // beams of a question: a warp
constexpr int kBeamMaxK = 64;
constexpr int kBcThreads = 256, kBcWarps = kBcThreads / 32, kBcPer = 16, kBcTile = kBcThreads * kBcPer;
constexpr int kBcCap = 1024;             // candidates of a tile that wait to be ranked

struct BeamRank { uint32_t key; int32_t idx; };      // float_to_key of the logit; equals: the lower index is better
__device__ __forceinline__ bool better(uint32_t ka, int ia, uint32_t kb, int ib) { return ka > kb || (ka == kb && ia < ib); }
constexpr uint32_t kNoKey = 0x007fffffu;              // float_to_key(-inf): no candidate at or below it (NaN never enters)

// A row's part: sum = sum exp(x - ref) over its logits (NaN: a logit was NaN or +inf), and its best logits in order.
struct BeamPart { double ref, sum; };

// The `want`-th best of a warp's lanes' (key, idx) pairs; key 0 where there are fewer candidates.
__device__ __forceinline__ BeamRank warp_nth(uint32_t key, int idx, int want) {
  BeamRank r{0u, 0x7fffffff};
  for (int i = 0; i < want; ++i) {
    r.key = __reduce_max_sync(0xffffffffu, key);
    if (r.key <= kNoKey) return {0u, 0x7fffffff};
    r.idx = __reduce_min_sync(0xffffffffu, key == r.key ? idx : 0x7fffffff);
    if (key == r.key && idx == r.idx) key = 0u;
  }
  return r;
}

__device__ __forceinline__ float ex2_part(float f) {      // |f| <= 1/2
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(f));
  return r;
}

template <typename T>
__global__ void __launch_bounds__(kBcThreads)
beam_rows_kernel(const T* __restrict__ logits, long long stride, const float* __restrict__ scores, int vocab, int splits, int tiles_per_split, int k,
                 BeamPart* __restrict__ parts, BeamRank* __restrict__ best) {
  __shared__ BeamRank s_list[2][kBeamMaxK], s_new[kBcCap], s_thr[kBcWarps];
  __shared__ uint32_t s_max[kBcWarps];
  __shared__ int s_count;
  __shared__ double s_sum[kBcWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long row = blockIdx.x / splits, part = blockIdx.x;
  const int t0 = (int)(blockIdx.x % splits) * tiles_per_split, v0 = t0 * kBcTile, v1 = (int)min((long long)vocab, (long long)v0 + (long long)tiles_per_split * kBcTile);
  const float score = scores[row];
  BeamRank* out = best + part * k;
  if (!(fabsf(score) < INFINITY) || v0 >= vocab) {           // a beam without a score offers nothing
    if (tid < k) out[tid] = {0u, 0x7fffffff};
    if (tid == 0) parts[part] = {0.0, 0.0};
    return;
  }
  const T* x_row = logits + row * stride;
  const int want = (k + kBcWarps - 1) / kBcWarps;
  int have = 0, cur = 0;                                    // entries of s_list[cur], in order
  BeamRank kth{kNoKey, 0x7fffffff};                         // what a newcomer has to beat
  uint32_t top = 0u;                                        // key of the largest logit so far
  float base = 0.f, big_n = 0.f;                            // the sum's reference: base + big_n * ln 2
  double ref = 0.0, sum = 0.0;
  bool nan = false;
  if (tid == 0) s_count = 0;
  for (int t = v0; t < v1; t += kBcTile) {
    float x[kBcPer];
#pragma unroll
    for (int j = 0; j < kBcPer; ++j) {
      const int i = t + j * kBcThreads + tid;
      x[j] = i < v1 ? to_f(x_row[i]) : -INFINITY;
    }
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < kBcPer; ++j) { m = fmaxf(m, x[j]); nan |= x[j] != x[j]; }
    const uint32_t key = float_to_key(m);
    // A lower bound of the tile's k best: each of the eight warps has `want` lanes whose best is at least the least of the warps'
    // want-th best.  It is a pair with an index, so that equal logits do not all pass.
    const uint32_t w_max = __reduce_max_sync(0xffffffffu, key);
    BeamRank thr{0u, 0x7fffffff};
    if (w_max > kth.key) {
      int at = 0;
#pragma unroll
      for (int j = kBcPer - 1; j >= 0; --j) if (x[j] == m) at = j;
      thr = warp_nth(key, t + at * kBcThreads + tid, want);
    }
    if (lane == 0) { s_max[warp] = w_max; s_thr[warp] = thr; }
    __syncthreads();
    uint32_t t_max = s_max[0];
    thr = s_thr[0];
#pragma unroll
    for (int w = 1; w < kBcWarps; ++w) {
      t_max = max(t_max, s_max[w]);
      if (better(thr.key, thr.idx, s_thr[w].key, s_thr[w].idx)) thr = s_thr[w];
    }
    if (t_max > top) {
      top = t_max;
      // The sum is kept relative to 2^big_n (times e^base for logits beyond 1e6): a power of two moves no bit of a term.
      const float mx = key_to_float(top);
      const float new_base = fabsf(mx) < 1e6f ? 0.f : mx, new_n = rintf((mx - new_base) * 1.44269504f);
      const double new_ref = (double)new_base + (double)new_n * 0.6931471805599453;
      if (sum != 0.0) sum *= exp(ref - new_ref);
      base = new_base; big_n = new_n; ref = new_ref;
    }
    if (key > kth.key) {
      if (t_max > kth.key) {
#pragma unroll
        for (int j = 0; j < kBcPer; ++j) {
          const uint32_t e = float_to_key(x[j]);
          const int i = t + j * kBcThreads + tid;
          if (x[j] == x[j] && e > kth.key && e >= thr.key && (e > thr.key || i <= thr.idx)) {
            const int at = atomicAdd(&s_count, 1);
            if (at < kBcCap) s_new[at] = {e, i};
          }
        }
      }
    }
    if (top > kNoKey) {
      // exp(x - base) / 2^big_n: the whole part of the exponent by integer arithmetic, the fraction (exact to 2^-25) by ex2.
      const float floor_x = key_to_float(top) - 80.f;         // below e^-80 of the largest: nothing in the sum's 53 bits
      float a = 0.f, b = 0.f;
#pragma unroll
      for (int j = 0; j < kBcPer; ++j) {
        const float y = fmaxf(x[j], floor_x) - base;
        const float r = fmaf(y, 1.44269504f, 12582912.f), n = r - 12582912.f;
        const float f = fmaf(y, 1.92596299e-8f, fmaf(y, 1.44269502f, -n));
        const float e = x[j] >= floor_x ? __int_as_float(__float_as_int(ex2_part(f)) + ((int)(n - big_n) << 23)) : 0.f;
        if (j & 1) b += e; else a += e;
      }
      sum += (double)(a + b);
    }
    __syncthreads();
    int n_new = s_count;
    if (n_new > kBcCap) {
      // Hardly ever: the warps' bests say little about the rest (a tile in which one warp's logits are all masked).  The k best
      // one at a time, each the best behind the one before.
      BeamRank last{0xffffffffu, -1};
      n_new = 0;
      while (n_new < k) {
        BeamRank mine{0u, 0x7fffffff};
#pragma unroll
        for (int j = 0; j < kBcPer; ++j) {
          const uint32_t e = float_to_key(x[j]);
          const int i = t + j * kBcThreads + tid;
          if (x[j] == x[j] && e > kth.key && better(last.key, last.idx, e, i) && better(e, i, mine.key, mine.idx)) mine = {e, i};
        }
        mine = warp_nth(mine.key, mine.idx, 1);
        if (lane == 0) s_thr[warp] = mine;
        __syncthreads();
        mine = s_thr[0];
#pragma unroll
        for (int w = 1; w < kBcWarps; ++w) if (better(s_thr[w].key, s_thr[w].idx, mine.key, mine.idx)) mine = s_thr[w];
        __syncthreads();
        if (mine.key == 0u) break;
        if (tid == 0) s_new[n_new] = mine;
        last = mine;
        ++n_new;
      }
      __syncthreads();
    }
    if (n_new > 0) {
      // Each entry's place is the number of better ones.
      const int all = have + n_new;
      for (int i = tid; i < all; i += kBcThreads) {
        const BeamRank mine = i < have ? s_list[cur][i] : s_new[i - have];
        int place = i < have ? i : 0;                         // the old ones are in order
        if (i >= have) for (int o = 0; o < have; ++o) place += better(s_list[cur][o].key, s_list[cur][o].idx, mine.key, mine.idx);
        for (int o = 0; o < n_new; ++o) place += better(s_new[o].key, s_new[o].idx, mine.key, mine.idx);
        if (place < k) s_list[cur ^ 1][place] = mine;
      }
      cur ^= 1;
      have = min(k, all);
      __syncthreads();
      if (have == k) kth = s_list[cur][k - 1];
      if (tid == 0) s_count = 0;
    }
  }
  if (tid < k) out[tid] = tid < have ? s_list[cur][tid] : BeamRank{0u, 0x7fffffff};
  nan = nan || top >= float_to_key(INFINITY);
  double s = nan ? __longlong_as_double(0x7ff8000000000000ll) : sum;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) s_sum[warp] = s;
  __syncthreads();
  if (tid == 0) {
    s = s_sum[0];
    for (int w = 1; w < kBcWarps; ++w) s += s_sum[w];
    parts[part] = {ref, s};
  }
}

// Order of 64-bit scores as integers.
__device__ __forceinline__ unsigned long long score_key(double v) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(v);
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ double key_score(unsigned long long k) {
  return __longlong_as_double((long long)(k >> 63 ? k & 0x7fffffffffffffffull : ~k));
}
// at: beam * vocab + token; key 0: none.  Equals go to the lower beam; within a beam, whose scores may be equal although its logits are
// not, to the larger logit, as in the choice of the row's best, and then to the lower token.
struct BeamScore { unsigned long long key; int32_t at; uint32_t logit; };
constexpr BeamScore kNoScore = {0ull, 0x7fffffff, 0u};
struct BeamOrder {
  int vocab;
  __device__ __forceinline__ bool operator()(const BeamScore& a, const BeamScore& b) const {
    if (a.key != b.key) return a.key > b.key;
    return a.logit != b.logit && a.at / vocab == b.at / vocab ? a.logit > b.logit : a.at < b.at;
  }
};
__device__ __forceinline__ BeamScore warp_best(BeamScore v, const BeamOrder& better) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    BeamScore w;
    w.key = __shfl_xor_sync(0xffffffffu, v.key, o);
    w.at = __shfl_xor_sync(0xffffffffu, v.at, o);
    w.logit = __shfl_xor_sync(0xffffffffu, v.logit, o);
    if (better(w, v)) v = w;
  }
  return v;
}

struct BeamChoiceOut { float* score; int32_t *beam, *token; float* live_score; int32_t *live_beam, *live_token; };

// One block per question.
__global__ void __launch_bounds__(kBcThreads)
beam_join_kernel(const BeamPart* __restrict__ parts, const BeamRank* __restrict__ best, const float* __restrict__ scores, int beams, int vocab,
                 int splits, int k, const int32_t* __restrict__ stop, int n_stop, const BeamChoiceOut out) {
  __shared__ double s_lse[kBeamMax], s_score[kBeamMax];
  __shared__ BeamScore s_new[kBcCap], s_thr[kBcWarps], s_done[kBeamMaxK];
  __shared__ int s_count;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long q = blockIdx.x;
  const BeamOrder better{vocab};
  if (tid == 0) s_count = 0;
  for (int b = warp; b < beams; b += kBcWarps) {
    const BeamPart* p = parts + (q * beams + b) * splits;
    double m = -INFINITY, s = 0.0;
    for (int i = lane; i < splits; i += 32) {
      const BeamPart v = p[i];
      if (v.sum != 0.0) {                                     // NaN too
        const double mx = fmax(m, v.ref);
        s = s * exp(m - mx) + v.sum * exp(v.ref - mx);
        m = mx;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double om = __shfl_xor_sync(0xffffffffu, m, o), os = __shfl_xor_sync(0xffffffffu, s, o), mx = fmax(m, om);
      if (mx > -INFINITY) s = s * exp(m - mx) + os * exp(om - mx);
      m = mx;
    }
    if (lane == 0) { s_lse[b] = m + log(s); s_score[b] = (double)scores[q * beams + b]; }    // nothing summed, or NaN: no candidates below
  }
  __syncthreads();
  const int per_row = splits * k, n = beams * per_row;
  auto candidate = [&](int c) -> BeamScore {
    const int b = c / per_row;
    const BeamRank r = best[(q * beams + b) * per_row + (c - b * per_row)];
    if (r.key <= kNoKey) return kNoScore;
    const double v = s_score[b] + ((double)key_to_float(r.key) - s_lse[b]);
    return v > -INFINITY && v < INFINITY ? BeamScore{score_key(v), b * vocab + r.idx, r.key} : kNoScore;
  };
  BeamScore mine = kNoScore;
  for (int c = tid; c < n; c += kBcThreads) {
    const BeamScore v = candidate(c);
    if (better(v, mine)) mine = v;
  }
  // As for a tile: the least of the warps' want-th best lanes bounds the k best from below.
  BeamScore thr = kNoScore;
  for (int i = 0, want = (k + kBcWarps - 1) / kBcWarps; i < want; ++i) {
    thr = warp_best(mine, better);
    if (mine.key == thr.key && mine.at == thr.at) mine = kNoScore;
  }
  if (lane == 0) s_thr[warp] = thr;
  __syncthreads();
  thr = s_thr[0];
  for (int w = 1; w < kBcWarps; ++w) if (better(thr, s_thr[w])) thr = s_thr[w];
  for (int c = tid; c < n; c += kBcThreads) {
    const BeamScore v = candidate(c);
    if (v.key && !better(thr, v)) {
      const int at = atomicAdd(&s_count, 1);
      if (at < kBcCap) s_new[at] = v;
    }
  }
  __syncthreads();
  int have = s_count;
  if (have > kBcCap) {                                        // hardly ever: one at a time
    BeamScore last{~0ull, -1, ~0u};
    for (have = 0; have < k; ++have) {
      mine = kNoScore;
      for (int c = tid; c < n; c += kBcThreads) {
        const BeamScore v = candidate(c);
        if (v.key && better(last, v) && better(v, mine)) mine = v;
      }
      mine = warp_best(mine, better);
      if (lane == 0) s_thr[warp] = mine;
      __syncthreads();
      mine = s_thr[0];
      for (int w = 1; w < kBcWarps; ++w) if (better(s_thr[w], mine)) mine = s_thr[w];
      __syncthreads();
      if (!mine.key) break;
      if (tid == 0) s_done[have] = mine;
      last = mine;
    }
  } else {
    for (int i = tid; i < have; i += kBcThreads) {
      const BeamScore v = s_new[i];
      int place = 0;
      for (int o = 0; o < have; ++o) place += better(s_new[o], v);
      if (place < k) s_done[place] = v;
    }
    have = min(have, k);
  }
  __syncthreads();
  if (tid < k) {
    const BeamScore v = s_done[tid];
    const bool on = tid < have;
    out.score[q * k + tid] = on ? (float)key_score(v.key) : -INFINITY;
    out.beam[q * k + tid] = on ? v.at / vocab : -1;
    out.token[q * k + tid] = on ? v.at % vocab : -1;
  }
  if (out.live_score && warp == 0) {
    int placed = 0;
    for (int c0 = 0; c0 < have; c0 += 32) {
      const int c = c0 + lane;
      bool on = c < have;
      const BeamScore v = on ? s_done[c] : BeamScore{0ull, 0, 0u};
      const int token = v.at % vocab;
      for (int i = 0; i < n_stop; ++i) on = on && stop[i] != token;
      const unsigned mask = __ballot_sync(0xffffffffu, on);
      const int place = placed + __popc(mask & ((1u << lane) - 1u));
      if (on && place < beams) {
        out.live_score[q * beams + place] = (float)key_score(v.key);
        out.live_beam[q * beams + place] = v.at / vocab;
        out.live_token[q * beams + place] = token;
      }
      placed += __popc(mask);
    }
    for (int i = placed + lane; i < beams; i += 32) {
      out.live_score[q * beams + i] = -INFINITY;
      out.live_beam[q * beams + i] = out.live_token[q * beams + i] = -1;
    }
  }
}

// ---------------------------------------------------------------------------------------------------- reordering
// What a slot holds of one tensor: everything (`bytes`), ring rows (of `bytes`, `rows` of them, the first `first` in front), or the half of
// two that the next position reads (of `bytes`).
constexpr int kReUnit = 4096, kReSearch = 4096;              // bytes a warp moves at a time; prefix sums kept in shared memory
struct ReorderCopy { int32_t src, dst, len, common; };
struct RingSpan { int c, n1, r0, n2; };                      // rows c .. c+n1-1, then n2 rows from r0 on, wrapping from the last row to `first`
__device__ __forceinline__ RingSpan ring_span(const msa_lm_state_part& s, const ReorderCopy& c) {
  RingSpan r;
  const int rows = (int)s.rows, turn = rows - s.first;
  r.c = c.common;
  r.n1 = max(0, min(s.first, c.len) - c.common);
  const int p0 = max(max(c.common, s.first), c.len - turn);
  r.n2 = turn > 0 ? max(0, c.len - p0) : 0;
  r.r0 = r.n2 ? ring_row(p0, s.first, rows) : 0;
  return r;
}
__device__ __forceinline__ long long part_bytes(const msa_lm_state_part& s, const ReorderCopy& c) {
  if (s.kind != MSA_LM_STATE_RING) return s.bytes;
  const RingSpan r = ring_span(s, c);
  return (long long)(r.n1 + r.n2) * s.bytes;
}

// One block: a warp per question decides who copies, then prefix sums of the copies' units.
__global__ void __launch_bounds__(1024)
reorder_plan_kernel(const int32_t* __restrict__ slot, const int32_t* __restrict__ parent, const int32_t* __restrict__ length,
                    const int32_t* __restrict__ shared, int batch, int beams, int n_slots, const msa_lm_state_part* __restrict__ part, int n_part,
                    int32_t* __restrict__ slot_out, int32_t* __restrict__ shared_out, ReorderCopy* __restrict__ copies, int32_t* __restrict__ off,
                    int32_t* __restrict__ count) {
  __shared__ int s_copies, s_part[32], s_run;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) s_copies = s_run = 0;
  __syncthreads();
  for (int e = warp; e < batch; e += 32) {
    const bool on = lane < beams;
    const int at = e * beams + lane;
    const int p = on ? parent[at] : -1, my_slot = on ? slot[at] : -1, len = max(0, length[e]);
    const bool valid = on && p >= 0 && p < beams;
    const unsigned named = __reduce_or_sync(0xffffffffu, valid ? 1u << p : 0u);
    const unsigned same = __match_any_sync(0xffffffffu, valid ? p : -1 - lane);
    const bool keeps = valid && lane == __ffs(same) - 1, needs = on && !keeps;
    const unsigned needy = __ballot_sync(0xffffffffu, needs);
    unsigned left = ~named & (beams == 32 ? ~0u : (1u << beams) - 1u);        // slots that nobody continues: as many as needy beams
    for (int i = __popc(needy & ((1u << lane) - 1u)); i > 0; --i) left &= left - 1u;
    const int from = keeps ? p : needs ? __ffs(left) - 1 : 0;                   // the beam whose slot this one takes
    const int to = __shfl_sync(0xffffffffu, my_slot, from), src = __shfl_sync(0xffffffffu, my_slot, valid ? p : 0);
    if (on) slot_out[at] = to;
    const bool copy = needs && valid && src >= 0 && src < n_slots && to >= 0 && to < n_slots && src != to;
    const unsigned mask = __ballot_sync(0xffffffffu, copy);
    int first = 0;
    if (lane == 0 && mask) first = atomicAdd(&s_copies, __popc(mask));
    first = __shfl_sync(0xffffffffu, first, 0);
    if (copy) {
      const int common = shared ? min(len, max(0, shared[((long long)e * beams + from) * beams + p])) : 0;
      copies[first + __popc(mask & ((1u << lane) - 1u))] = {src, to, len, common};
    }
    if (shared_out) {
      const int origin = valid ? p : from;
      for (int i = 0; i < beams; ++i) {
        const int other = __shfl_sync(0xffffffffu, origin, i);
        if (on) shared_out[((long long)e * beams + i) * beams + lane] = other == origin ? len : shared[((long long)e * beams + other) * beams + origin];
      }
    }
  }
  __syncthreads();
  const int n = s_copies * n_part;
  for (int i0 = 0; i0 < n; i0 += 1024) {
    const int i = i0 + (int)threadIdx.x;
    int u = 0;
    if (i < n) u = (int)((part_bytes(part[i % n_part], copies[i / n_part]) + kReUnit - 1) / kReUnit);
    int run = u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, run, o); if (lane >= o) run += v; }
    if (lane == 31) s_part[warp] = run;
    __syncthreads();
    int before = s_run;
    for (int w = 0; w < warp; ++w) before += s_part[w];
    if (i < n) off[i] = before + run - u;
    __syncthreads();
    if (threadIdx.x == 1023) s_run = before + run;
    __syncthreads();
  }
  if (threadIdx.x == 0) { off[n] = s_run; *count = n; }
}

template <typename V>
__device__ __forceinline__ void move_bytes(const unsigned char* src, unsigned char* dst, long long b0, long long b1, const long long (&end)[2],
                                           const long long (&add)[3], int lane) {
  constexpr int kAhead = 8;
  for (long long b = b0 + lane * (int)sizeof(V); b < b1; b += 32 * kAhead * (int)sizeof(V)) {
    V v[kAhead];
    long long at[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const long long o = b + u * 32 * (int)sizeof(V);
      at[u] = o + (o < end[0] ? add[0] : o < end[1] ? add[1] : add[2]);
      if (o < b1) v[u] = *reinterpret_cast<const V*>(src + at[u]);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (b + u * 32 * (int)sizeof(V) < b1) *reinterpret_cast<V*>(dst + at[u]) = v[u];
  }
}

// Every warp takes an equal run of the units.
__global__ void __launch_bounds__(256)
reorder_copy_kernel(const msa_lm_state_part* part, int n_part, const ReorderCopy* copies, const int32_t* off, const int32_t* count) {
  __shared__ int32_t s_off[kReSearch];
  grid_dependency_wait();
  const int n = *count;
  const bool near = n + 1 <= kReSearch;
  if (near) {
    for (int i = threadIdx.x; i <= n; i += 256) s_off[i] = off[i];
    __syncthreads();
  }
  const int32_t* at = near ? s_off : off;
  const int lane = threadIdx.x & 31;
  const long long units = at[n], w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5), n_w = (long long)gridDim.x * 8;
  const long long u1 = units * (w + 1) / n_w;
  long long u = units * w / n_w;
  if (u >= u1) return;
  int i = owner_of(at, n, (int)u);
  while (u < u1) {
    while (at[i + 1] <= u) ++i;                              // parts of which nothing moves have no units
    const ReorderCopy c = copies[i / n_part];
    const msa_lm_state_part s = part[i % n_part];
    long long total = s.bytes, end[2] = {total, total}, add[3] = {0, 0, 0};
    if (s.kind == MSA_LM_STATE_RING) {
      const RingSpan r = ring_span(s, c);
      total = (long long)(r.n1 + r.n2) * s.bytes;
      end[0] = (long long)r.n1 * s.bytes;
      end[1] = end[0] + (long long)min(r.n2, (int)s.rows - r.r0) * s.bytes;
      add[0] = (long long)r.c * s.bytes;
      add[1] = (long long)r.r0 * s.bytes - end[0];
      add[2] = (long long)s.first * s.bytes - end[1];
    } else if (s.kind == MSA_LM_STATE_HALF) {
      add[0] = add[1] = add[2] = (long long)(c.len & 1) * s.bytes;
    }
    const unsigned char* src = reinterpret_cast<const unsigned char*>(s.base) + c.src * s.slot_bytes;
    unsigned char* dst = reinterpret_cast<unsigned char*>(s.base) + c.dst * s.slot_bytes;
    const long long last = min(u1, (long long)at[i + 1]);
    const long long b0 = (u - at[i]) * kReUnit, b1 = min(total, (last - at[i]) * kReUnit);
    if (s.align >= 16) move_bytes<uint4>(src, dst, b0, b1, end, add, lane);
    else if (s.align >= 4) move_bytes<uint32_t>(src, dst, b0, b1, end, add, lane);
    else move_bytes<uint16_t>(src, dst, b0, b1, end, add, lane);
    u = last;
  }
}

template <typename T>
void launch_beam_rows(const void* logits, int64_t stride, const float* scores, int64_t rows, int vocab, int splits, int tiles_per_split, int k,
                      BeamPart* parts, BeamRank* best, cudaStream_t st) {
  beam_rows_kernel<T><<<(unsigned)(rows * splits), kBcThreads, 0, st>>>((const T*)logits, stride, scores, vocab, splits, tiles_per_split, k, parts, best);
}

}  // namespace msa

using namespace msa;

// Parts of a row: four blocks an SM, each of whole tiles.
static int beam_splits(int64_t rows, int32_t vocab, int* tiles_per_split) {
  const int tiles = (vocab + kBcTile - 1) / kBcTile;
  const int64_t want = (148 * 4 + rows - 1) / rows;
  const int splits = (int)(want < tiles ? want : tiles);
  *tiles_per_split = (tiles + splits - 1) / splits;
  return (tiles + *tiles_per_split - 1) / *tiles_per_split;
}

extern "C" int64_t msa_lm_beam_topk_workspace(int32_t batch, int32_t beams, int32_t vocab, int32_t k) {
  if (batch <= 0 || beams <= 0 || vocab <= 0 || k <= 0) return 0;
  int per = 0;
  const int64_t parts = (int64_t)batch * beams * beam_splits((int64_t)batch * beams, vocab, &per);
  return parts * ((int64_t)sizeof(BeamPart) + (int64_t)k * (int64_t)sizeof(BeamRank));
}

extern "C" int msa_lm_beam_topk(const void* logits, int64_t stride, int32_t dtype, const float* scores, int32_t batch, int32_t beams, int32_t vocab,
                                int32_t k, const int32_t* stop, int32_t n_stop, void* workspace, float* score, int32_t* beam, int32_t* token,
                                float* live_score, int32_t* live_beam, int32_t* live_token, void* stream) {
  MSA_REQUIRE(dtype_ok(dtype) && batch >= 0 && beams >= 1 && beams <= kBeamMax && vocab >= 1 && (int64_t)beams * vocab < (1ll << 31) - 2 * kBcTile && stride >= 0,
              "beam_topk: bad dtype or sizes (1 to %d beams)", kBeamMax);
  MSA_REQUIRE(k >= 1 && k <= kBeamMaxK && (int64_t)k <= (int64_t)beams * vocab, "beam_topk: k must be 1 to %d and no more than there are candidates", kBeamMaxK);
  if (batch == 0) return MSA_OK;
  MSA_REQUIRE(logits && scores && workspace && score && beam && token, "beam_topk: null pointer");
  MSA_REQUIRE(n_stop >= 0 && (n_stop == 0 || stop) && (live_score != nullptr) == (live_beam != nullptr) && (live_score != nullptr) == (live_token != nullptr),
              "beam_topk: stop tokens or live outputs missing");
  MSA_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 8 == 0, "beam_topk: workspace must be 8-byte aligned");
  const int64_t rows = (int64_t)batch * beams;
  int per = 0;
  const int splits = beam_splits(rows, vocab, &per);
  MSA_REQUIRE(rows * splits < (1ll << 31), "beam_topk: too many rows");
  BeamPart* parts = (BeamPart*)workspace;
  BeamRank* best = (BeamRank*)(parts + rows * splits);
  cudaStream_t st = (cudaStream_t)stream;
  MSA_LM_DISPATCH(dtype, { launch_beam_rows<T>(logits, stride, scores, rows, vocab, splits, per, k, parts, best, st); });
  MSA_LAUNCH_OK("beam_rows_kernel");
  const BeamChoiceOut out{score, beam, token, live_score, live_beam, live_token};
  beam_join_kernel<<<(unsigned)batch, kBcThreads, 0, st>>>(parts, best, scores, beams, vocab, splits, k, stop, n_stop, out);
  MSA_LAUNCH_OK("beam_join_kernel");
  return MSA_OK;
}

extern "C" int64_t msa_lm_reorder_workspace(int32_t batch, int32_t beams, int32_t n_part) {
  if (batch <= 0 || beams <= 0 || n_part <= 0) return 0;
  const int64_t n = (int64_t)batch * beams;
  return n * (int64_t)sizeof(ReorderCopy) + (n * n_part + 2) * 4;
}

extern "C" int msa_lm_reorder(const int32_t* slot, const int32_t* parent, const int32_t* length, const int32_t* shared, int32_t batch, int32_t beams,
                              int32_t n_slots, const msa_lm_state_part* parts, int32_t n_part, int32_t* slot_out, int32_t* shared_out, void* workspace,
                              void* stream) {
  MSA_REQUIRE(batch >= 0 && beams >= 1 && beams <= kBeamMax && n_slots >= 1 && n_part >= 1, "reorder: bad sizes (1 to %d beams)", kBeamMax);
  if (batch == 0) return MSA_OK;
  MSA_REQUIRE(slot && parent && length && parts && slot_out && workspace && (shared_out == nullptr || shared), "reorder: null pointer");
  MSA_REQUIRE(slot_out != slot && (shared_out == nullptr || shared_out != shared), "reorder: the new tables must not be the old ones");
  MSA_REQUIRE((int64_t)batch * beams * n_part < (1ll << 31) - 2, "reorder: too many beams and parts");
  MSA_REQUIRE(aligned16(workspace), "reorder: workspace must be 16-byte aligned");
  const int64_t n = (int64_t)batch * beams;
  ReorderCopy* copies = (ReorderCopy*)workspace;
  int32_t* off = (int32_t*)(copies + n);
  int32_t* count = off + n * n_part + 1;
  cudaStream_t st = (cudaStream_t)stream;
  reorder_plan_kernel<<<1, 1024, 0, st>>>(slot, parent, length, shared, batch, beams, n_slots, parts, n_part, slot_out, shared_out, copies, off, count);
  MSA_LAUNCH_OK("reorder_plan_kernel");
  int n_sm = 0;
  MSA_OK_OR_RETURN(device_sm_count(&n_sm));
  MSA_CUDA_OK(launch_kernel_pdl(reorder_copy_kernel, dim3((unsigned)(8 * n_sm)), dim3(256), 0, st, true, parts, n_part, (const ReorderCopy*)copies,
                                (const int32_t*)off, (const int32_t*)count));
  MSA_LAUNCH_OK("reorder_copy_kernel");
  return MSA_OK;
}
