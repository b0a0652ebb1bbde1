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
constexpr int kBcCap = 1024;             // entries of a part that wait to be ranked
constexpr int kBjThreads = 512, kBjWarps = kBjThreads / 32;

// A logit and its token as one number: the larger logit is better, of equals the lower token.  0: none; NaN and -inf never enter.
typedef unsigned long long Rank;
constexpr uint32_t kNoKey = 0x007fffffu;              // float_to_key(-inf)
__device__ __forceinline__ Rank rank_of(float x, int idx) { return (Rank)float_to_key(x + 0.f) << 32 | (uint32_t)~idx; }   // -0 is 0
__device__ __forceinline__ uint32_t rank_key(Rank r) { return (uint32_t)(r >> 32); }
__device__ __forceinline__ int rank_idx(Rank r) { return (int)~(uint32_t)r; }

// A row's part: the sum of e^x over its logits as sum * 2^n * e^base (NaN: a logit was NaN or +inf).
struct BeamPart { double sum; int32_t n; float base; };

// p += v.
__device__ __forceinline__ double pow2(float e) { return e < -1000.f ? 0.0 : __longlong_as_double((long long)((int)e + 1023) << 52); }   // whole e <= 0
__device__ __forceinline__ void join_sums(BeamPart& p, const BeamPart& v) {
  if (v.sum == 0.0) return;
  if (p.sum == 0.0) { p = v; return; }
  if (p.base == 0.f && v.base == 0.f) {
    const int n = max(p.n, v.n);
    p.sum = p.sum * pow2((float)(p.n - n)) + v.sum * pow2((float)(v.n - n));
    p.n = n;
    return;
  }
  const double rp = (double)p.base + p.n * 0.6931471805599453, rv = (double)v.base + v.n * 0.6931471805599453;
  if (rp >= rv) { p.sum += v.sum * exp(rv - rp); return; }
  const double mine = p.sum * exp(rp - rv);
  p = v;
  p.sum += mine;
}

__device__ __forceinline__ BeamPart other_part(const BeamPart& p, int o) {
  return {__shfl_xor_sync(0xffffffffu, p.sum, o), __shfl_xor_sync(0xffffffffu, p.n, o), __shfl_xor_sync(0xffffffffu, p.base, o)};
}

// The `want`-th best of a warp's lanes, each with one entry; 0 where there are fewer.
__device__ __forceinline__ Rank warp_nth(Rank mine, int want) {
  uint32_t key = 0u, low = 0u;
  for (int i = 0; i < want; ++i) {
    key = __reduce_max_sync(0xffffffffu, rank_key(mine));
    if (key <= kNoKey) return 0ull;
    low = __reduce_max_sync(0xffffffffu, rank_key(mine) == key ? (uint32_t)mine : 0u);
    if (mine == ((Rank)key << 32 | low)) mine = 0ull;
  }
  return (Rank)key << 32 | low;
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float ex2_part(float f) {      // |f| <= 1/2
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(f));
  return r;
}

template <typename T>
__device__ __forceinline__ void load_tile(const T* x_row, int t, int v1, float (&x)[kBcPer]) {
  if (t + kBcTile <= v1) {
#pragma unroll
    for (int j = 0; j < kBcPer; ++j) x[j] = to_f(x_row[t + j * kBcThreads + (int)threadIdx.x]);
  } else {
#pragma unroll
    for (int j = 0; j < kBcPer; ++j) {
      const int i = t + j * kBcThreads + (int)threadIdx.x;
      x[j] = i < v1 ? to_f(x_row[i]) : -INFINITY;
    }
  }
}

struct BeamScratch { Rank list[2][kBeamMaxK], fresh[kBcCap], post[kBcWarps]; int count; };

// Entries 0 .. n-1 of s.fresh join the `have` of s.list[cur], which are in order: each one's place is the number of better ones.
__device__ __forceinline__ void rank_entries(BeamScratch& s, int n, int k, int& have, int& cur) {
  for (int i = threadIdx.x; i < have + n; i += kBcThreads) {
    const Rank mine = i < have ? s.list[cur][i] : s.fresh[i - have];
    int place = i < have ? i : 0;
    if (i >= have) for (int o = 0; o < have; ++o) place += s.list[cur][o] > mine;
#pragma unroll 4
    for (int o = 0; o < n; ++o) place += s.fresh[o] > mine;
    if (place < k) s.list[cur ^ 1][place] = mine;
  }
  cur ^= 1;
  have = min(k, have + n);
  __syncthreads();
}

// The k best of a part whatever its order, tile by tile, where too many entries passed the bound on the way (rows that rise towards their
// end, masks that leave a warp without logits): 64 beams over 12,345 sorted logits take 1.7 times as long as unsorted ones.
template <typename T>
__device__ __noinline__ int ordered_best(const T* x_row, int v0, int v1, int k, BeamScratch& s) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, want = (k + kBcWarps - 1) / kBcWarps;
  int have = 0, cur = 0;
  Rank kth = 0ull;                                          // what a newcomer has to beat
  for (int t = v0; t < v1; t += kBcTile) {
    float x[kBcPer];
    load_tile(x_row, t, v1, x);
    Rank best = 0ull;
#pragma unroll
    for (int j = 0; j < kBcPer; ++j) {
      const Rank e = rank_of(x[j], t + j * kBcThreads + (int)threadIdx.x);
      if (x[j] > -INFINITY && e > best) best = e;
    }
    const Rank post = warp_nth(best, want);
    __syncthreads();
    if (lane == 0) s.post[warp] = post;
    if (threadIdx.x == 0) s.count = 0;
    __syncthreads();
    Rank bound = s.post[0];
#pragma unroll
    for (int w = 1; w < kBcWarps; ++w) bound = min(bound, s.post[w]);
#pragma unroll
    for (int j = 0; j < kBcPer; ++j) {
      const Rank e = rank_of(x[j], t + j * kBcThreads + (int)threadIdx.x);
      if (x[j] > -INFINITY && e > kth && e >= bound) {
        const int at = atomicAdd(&s.count, 1);
        if (at < kBcCap) s.fresh[at] = e;
      }
    }
    __syncthreads();
    int n = s.count;
    if (n > kBcCap) {                                       // the bound says nothing: one at a time, each the best behind the one before
      Rank last = ~0ull;
      for (n = 0; n < k; ++n) {
        best = 0ull;
#pragma unroll
        for (int j = 0; j < kBcPer; ++j) {
          const Rank e = rank_of(x[j], t + j * kBcThreads + (int)threadIdx.x);
          if (x[j] > -INFINITY && e > kth && e < last && e > best) best = e;
        }
        best = warp_nth(best, 1);
        __syncthreads();
        if (lane == 0) s.post[warp] = best;
        __syncthreads();
        last = s.post[0];
#pragma unroll
        for (int w = 1; w < kBcWarps; ++w) last = max(last, s.post[w]);
        if (last == 0ull) break;
        if (threadIdx.x == 0) s.fresh[n] = last;
      }
      __syncthreads();
    }
    rank_entries(s, n, k, have, cur);
    if (have == k) kth = s.list[cur][k - 1];
  }
  if (cur) {
    for (int i = threadIdx.x; i < have; i += kBcThreads) s.list[0][i] = s.list[1][i];
    __syncthreads();
  }
  return have;
}

// One block per part of a row.  Its warps walk the part's tiles without waiting for one another: each keeps its lanes' best logits and
// publishes the want-th of them, want = ceil(k / 8), so that the least of the eight is a bound that k logits reach; what reaches it is
// set aside, some 2.5 k (1 + log tiles) entries, and ranked at the end.  The next tile's loads are in flight meanwhile.
template <typename T>
__global__ void __launch_bounds__(kBcThreads, 3)
beam_rows_kernel(const T* __restrict__ logits, long long stride, const float* __restrict__ scores, int vocab, int splits, int tiles_per_split, int k,
                 BeamPart* __restrict__ parts, Rank* __restrict__ best) {
  __shared__ BeamScratch s;
  __shared__ double s_sum[kBcWarps];
  __shared__ int s_n[kBcWarps];
  __shared__ float s_base[kBcWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long row = blockIdx.x / splits, part = blockIdx.x;
  const int v0 = (int)(blockIdx.x % splits) * tiles_per_split * kBcTile, v1 = (int)min((long long)vocab, (long long)v0 + (long long)tiles_per_split * kBcTile);
  Rank* out = best + part * k;
  if (!(fabsf(scores[row]) < INFINITY)) {                    // a beam without a score offers nothing
    if (tid < k) out[tid] = 0ull;
    if (tid == 0) parts[part] = {0.0, 0, 0.f};
    return;
  }
  const T* x_row = logits + row * stride;
  const int want = (k + kBcWarps - 1) / kBcWarps;
  float x[kBcPer];
  load_tile(x_row, v0, v1, x);
  if (tid == 0) s.count = 0;
  float mine = -INFINITY;                                   // this lane's best, its token, and the warp's best
  int mine_at = 0;
  uint32_t top = 0u;
  float base = 0.f, big_n = 0.f;                            // the warp's reference
  double sum = 0.0;
  bool nan = false;
  for (int t = v0; t < v1; t += kBcTile) {
    float nx[kBcPer];
    if (t + kBcTile < v1) load_tile(x_row, t + kBcTile, v1, nx);
    float m = x[0], m2 = x[1];
#pragma unroll
    for (int j = 2; j < kBcPer; j += 2) { m = max_nan(m, x[j]); m2 = max_nan(m2, x[j + 1]); }
    m = max_nan(m, m2);
    if (m != m) {                                           // the maximum that passes over NaN
      nan = true;
      m = -INFINITY;
#pragma unroll
      for (int j = 0; j < kBcPer; ++j) m = fmaxf(m, x[j]);
    }
    if (__any_sync(0xffffffffu, m > mine)) {
      if (m > mine) {
        mine = m;
#pragma unroll
        for (int j = kBcPer - 1; j >= 0; --j) if (x[j] == m) mine_at = t + j * kBcThreads + tid;
      }
      const Rank post = warp_nth(mine > -INFINITY ? rank_of(mine, mine_at) : 0ull, want);
      if (lane == 0) *(volatile Rank*)&s.post[warp] = post;
      const uint32_t t_max = __reduce_max_sync(0xffffffffu, float_to_key(m));
      if (t_max > top) {
        // The sum is kept relative to a power of two, which moves no bit of a term (and to e^base for logits beyond 1e6).
        const float mx = key_to_float(t_max), new_base = fabsf(mx) < 1e6f ? 0.f : mx, new_n = rintf((mx - new_base) * 1.44269504f);
        if (sum != 0.0) sum *= new_base == 0.f && base == 0.f ? pow2(big_n - new_n) : exp(((double)base - new_base) + ((double)big_n - new_n) * 0.6931471805599453);
        top = t_max; base = new_base; big_n = new_n;
      }
    } else if (t == v0 && lane == 0) {
      s.post[warp] = 0ull;                                  // nothing but -inf
    }
    if (t == v0) __syncthreads();                           // later a bound that is behind lets a few more pass
    Rank bound = *(volatile Rank*)&s.post[0];
#pragma unroll
    for (int w = 1; w < kBcWarps; ++w) bound = min(bound, *(volatile Rank*)&s.post[w]);
    const float least = rank_key(bound) > kNoKey ? key_to_float(rank_key(bound)) : -INFINITY;
    if (m >= least) {
#pragma unroll
      for (int j = 0; j < kBcPer; ++j)
        if (x[j] >= least) {
          const Rank e = rank_of(x[j], t + j * kBcThreads + tid);
          if (e >= bound && x[j] > -INFINITY) {
            const int at = atomicAdd(&s.count, 1);
            if (at < kBcCap) s.fresh[at] = e;
          }
        }
    }
    if (top > kNoKey) {
      // e^x / 2^big_n: the exponent's whole part by integer arithmetic, the fraction (exact to 2^-25) by ex2.
      const float floor_x = key_to_float(top) - 80.f, magic = 12582912.f - big_n;
      float a = 0.f, b = 0.f;
      if (base == 0.f) {
#pragma unroll
        for (int j = 0; j < kBcPer; ++j) {
          const float y = fmaxf(x[j], floor_x);             // e^-80 of the largest is nothing in the sum's 53 bits, and -inf may count as that
          const float r = fmaf(y, 1.44269504f, magic), f = fmaf(y, 1.92596299e-8f, fmaf(y, 1.44269502f, magic - r));
          const float e = __int_as_float(__float_as_int(ex2_part(f)) + (__float_as_int(r) << 23));
          if (j & 1) b += e; else a += e;
        }
      } else {                                              // big_n is 0
#pragma unroll
        for (int j = 0; j < kBcPer; ++j) a += x[j] >= floor_x ? expf(x[j] - base) : 0.f;
      }
      sum += (double)(a + b);
    }
#pragma unroll
    for (int j = 0; j < kBcPer; ++j) x[j] = nx[j];
  }
  if (nan || top >= float_to_key(INFINITY)) sum = __longlong_as_double(0x7ff8000000000000ll);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) { s_sum[warp] = sum; s_n[warp] = (int)big_n; s_base[warp] = base; }
  __syncthreads();
  int n = s.count, have = 0, cur = 0;
  if (n > kBcCap) {
    have = ordered_best(x_row, v0, v1, k, s);
  } else {
    // What reaches the bound of all tiles is what remains: every thread holds up to four of the entries meanwhile.
    Rank bound = s.post[0], keep[kBcCap / kBcThreads];
#pragma unroll
    for (int w = 1; w < kBcWarps; ++w) bound = min(bound, s.post[w]);
#pragma unroll
    for (int i = 0; i < kBcCap / kBcThreads; ++i) keep[i] = i * kBcThreads + tid < n ? s.fresh[i * kBcThreads + tid] : 0ull;
    __syncthreads();
    if (tid == 0) s.count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBcCap / kBcThreads; ++i) if (keep[i] != 0ull && keep[i] >= bound) s.fresh[atomicAdd(&s.count, 1)] = keep[i];
    __syncthreads();
    rank_entries(s, s.count, k, have, cur);
  }
  if (tid < k) out[tid] = tid < have ? s.list[cur][tid] : 0ull;
  if (warp == kBcWarps - 1) {
    BeamPart p = {s_sum[lane % kBcWarps], s_n[lane % kBcWarps], s_base[lane % kBcWarps]};
#pragma unroll
    for (int o = 1; o < kBcWarps; o <<= 1) join_sums(p, other_part(p, o));
    if (lane == 0) parts[part] = p;
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

// One block per question.  Scores are 64-bit; a bound from below, in 32 bits rounded down, leaves a few times k candidates to rank.
__global__ void __launch_bounds__(kBjThreads)
beam_join_kernel(const BeamPart* parts, const Rank* best, const float* scores, int beams, int vocab, int splits, int k, const int32_t* stop, int n_stop,
                 const BeamChoiceOut out) {
  grid_dependency_wait();
  __shared__ BeamPart s_part[kBeamMax];
  __shared__ double s_lse[kBeamMax], s_score[kBeamMax];
  __shared__ BeamScore s_new[kBcCap], s_one[kBjWarps], s_done[kBeamMaxK];
  __shared__ uint32_t s_post[kBjWarps];
  __shared__ int s_count;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long q = blockIdx.x;
  const BeamOrder better{vocab};
  if (tid == 0) s_count = 0;
  for (int b = warp; b < beams; b += kBjWarps) {
    BeamPart p = {0.0, 0, 0.f};
    for (int i = lane; i < splits; i += 32) join_sums(p, parts[(q * beams + b) * splits + i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) join_sums(p, other_part(p, o));
    if (lane == 0) s_part[b] = p;
  }
  __syncthreads();
  if (tid < beams) {                                          // nothing summed, or NaN: no candidates below
    const BeamPart p = s_part[tid];
    s_lse[tid] = ((double)p.base + (double)p.n * 0.6931471805599453) + log(p.sum);
    s_score[tid] = (double)scores[q * beams + tid];
  }
  __syncthreads();
  // Candidates are taken the parts' best ones first, so that every warp sees some of those.
  const int lists = beams * splits, n = lists * k;
  const Rank* ranks = best + q * n;
  auto candidate = [&](int c) -> BeamScore {
    const int place = c / lists, list = c - place * lists, b = list / splits;
    const Rank r = ranks[list * k + place];
    if (r == 0ull) return kNoScore;
    const double v = s_score[b] + ((double)key_to_float(rank_key(r)) - s_lse[b]);
    return v > -INFINITY && v < INFINITY ? BeamScore{score_key(v), b * vocab + rank_idx(r), rank_key(r)} : kNoScore;
  };
  unsigned long long top = 0ull;
  for (int c = tid; c < n; c += kBjThreads) top = max(top, candidate(c).key);
  uint32_t key = top ? float_to_key(__double2float_rd(key_score(top))) : 0u, post = 0u;
  const int warps = min(kBjWarps, (n + 31) / 32);               // those with candidates: each has `want` that reach the bound
  for (int i = 0, want = (k + warps - 1) / warps; i < want; ++i) {
    post = __reduce_max_sync(0xffffffffu, key);
    const unsigned who = __ballot_sync(0xffffffffu, key == post);
    if (lane == __ffs(who) - 1) key = 0u;
  }
  if (lane == 0) s_post[warp] = post;
  __syncthreads();
  uint32_t bound = s_post[0];
  for (int w = 1; w < warps; ++w) bound = min(bound, s_post[w]);
  const unsigned long long least = bound ? score_key((double)key_to_float(bound)) : 1ull;
  for (int c = tid; c < n; c += kBjThreads) {
    const BeamScore v = candidate(c);
    if (v.key >= least) {
      const int at = atomicAdd(&s_count, 1);
      if (at < kBcCap) s_new[at] = v;
    }
  }
  __syncthreads();
  int have = s_count;
  if (have > kBcCap) {                                        // equal scores by the hundred: one at a time
    BeamScore last{~0ull, -1, ~0u};
    for (have = 0; have < k; ++have) {
      BeamScore mine = kNoScore;
      for (int c = tid; c < n; c += kBjThreads) {
        const BeamScore v = candidate(c);
        if (v.key && better(last, v) && better(v, mine)) mine = v;
      }
      mine = warp_best(mine, better);
      if (lane == 0) s_one[warp] = mine;
      __syncthreads();
      mine = s_one[0];
      for (int w = 1; w < kBjWarps; ++w) if (better(s_one[w], mine)) mine = s_one[w];
      __syncthreads();
      if (!mine.key) break;
      if (tid == 0) s_done[have] = mine;
      last = mine;
    }
  } else {
    for (int i = tid; i < have; i += kBjThreads) {
      const BeamScore v = s_new[i];
      int place = 0;
#pragma unroll 4
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
                      BeamPart* parts, Rank* best, cudaStream_t st) {
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
  return parts * ((int64_t)sizeof(BeamPart) + (int64_t)k * (int64_t)sizeof(Rank));
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
  Rank* best = (Rank*)(parts + rows * splits);
  cudaStream_t st = (cudaStream_t)stream;
  MSA_LM_DISPATCH(dtype, { launch_beam_rows<T>(logits, stride, scores, rows, vocab, splits, per, k, parts, best, st); });
  MSA_LAUNCH_OK("beam_rows_kernel");
  const BeamChoiceOut out{score, beam, token, live_score, live_beam, live_token};
  MSA_CUDA_OK(launch_kernel_pdl(beam_join_kernel, dim3((unsigned)batch), dim3(kBjThreads), 0, st, true, parts, best, scores, beams, vocab, splits, k, stop,
                                n_stop, out));
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
