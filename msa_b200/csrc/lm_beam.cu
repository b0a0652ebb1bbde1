// Beam search: the choice of the next beams from the logits, and the reordering of the sequence states that follows from it.
//
// Choice.  A candidate (beam b, token t) has the score  s_b + (x_bt - lse_b),  lse_b = log sum_t exp x_bt.  Within a row the order is
// that of the logits, so one pass over a row yields its sum and the largest logit of every 512, and a question's k best lie in the k chunks
// whose largest are the best; the second kernel ranks those, reads them again and ranks what lies in them: scores are added and compared in
// 64 bits, a row's sum (terms of 2^-22, added by sixteen in 32 bits, from there on in 64) is good to 5.5e-7 of itself.  Its last bits depend on the
// number of parts that the rows are cut into, and so on how many rows there are.  Bound by the one read
// of the logits (48 x 4 rows of 151,936 fp32: 23 us at 5.1 TB/s, then 8), for few rows by the second kernel's chain of barriers (7 us).
//
// Reordering.  New beam j continues beam parent[j].  Its first child keeps a beam's slot, the others take slots that nobody
// continues: sources and destinations never meet, and no second buffer is needed.  Bound by the copied bytes, read and written once.
#include "lm_common.cuh"
#include "tc_attn_common.cuh"

namespace msa {

constexpr int kBeamMax = 32;             // beams of a question: a warp
constexpr int kBeamMaxK = 64;
constexpr int kBcThreads = 256, kBcWarps = kBcThreads / 32, kBcPer = 16, kBcTile = kBcThreads * kBcPer, kBcBlocks = 4;
constexpr int kBcChunk = 32 * kBcPer;    // logits of a warp's turn, consecutive ones
constexpr int kBjThreads = 512, kBjWarps = kBjThreads / 32, kBjHold = 4;
constexpr int kBjCap = 1024;             // entries that wait to be ranked

// A row's part: the sum of e^x over its logits as sum * 2^n * e^base (NaN: a logit was NaN or +inf).
struct BeamPart { double sum; int32_t n; float base; };

__device__ __forceinline__ double pow2(float e) { return e < -1000.f ? 0.0 : __longlong_as_double((long long)((int)e + 1023) << 52); }   // whole e <= 0
__device__ __noinline__ double exp_of(double v) { return exp(v); }                     // hardly ever called
// p += v.
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
  if (rp >= rv) { p.sum += v.sum * exp_of(rv - rp); return; }
  const double mine = p.sum * exp_of(rp - rv);
  p = v;
  p.sum += mine;
}
__device__ __forceinline__ BeamPart other_part(const BeamPart& p, int o) {
  return {__shfl_xor_sync(0xffffffffu, p.sum, o), __shfl_xor_sync(0xffffffffu, p.n, o), __shfl_xor_sync(0xffffffffu, p.base, o)};
}

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The logits of a warp's turn: lane by lane, so that a row may start anywhere and is summed in the same order wherever it does.
template <typename T>
__device__ __forceinline__ void load_chunk(const T* x_row, int i0, int v1, float (&x)[kBcPer]) {
  const int lane = threadIdx.x & 31;
  if (i0 + kBcChunk <= v1) {
#pragma unroll
    for (int j = 0; j < kBcPer; ++j) x[j] = to_f(x_row[i0 + j * 32 + lane]);
  } else {
#pragma unroll
    for (int j = 0; j < kBcPer; ++j) x[j] = i0 + j * 32 + lane < v1 ? to_f(x_row[i0 + j * 32 + lane]) : -INFINITY;
  }
}

// One pass over the logits: every row's sum, and the largest logit of every 512.  The k best of a question lie in the k chunks with the
// best largest logits (any other chunk has k logits above its own largest, or equal and at lower tokens), so nothing else is kept:
// ranking on the way, by bounds from what the block had seen, took 45 us for 48 x 4 rows of 151,936 where this takes 22.  The loads of a warp's
// next chunk are in flight while it works on one.
template <typename T>
__global__ void __launch_bounds__(kBcThreads, kBcBlocks)
beam_rows_kernel(const T* __restrict__ logits, long long stride, const float* __restrict__ scores, int vocab, int chunks, int splits, int tiles_per_split,
                 BeamPart* __restrict__ parts, float* __restrict__ largest) {
  __shared__ BeamPart s_part[kBcWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = blockIdx.x / splits, part = blockIdx.x;
  const int v0 = (int)(blockIdx.x % splits) * tiles_per_split * kBcTile, v1 = (int)min((long long)vocab, (long long)v0 + (long long)tiles_per_split * kBcTile);
  float* out = largest + row * chunks;
  const T* x_row = logits + row * stride;
  const bool live = fabsf(scores[row]) < INFINITY;            // a beam without a score offers nothing
  float top = -INFINITY, base = 0.f, big_n = 0.f, floor_x = 0.f;   // the warp's largest logit, its sum's reference, and what vanishes beside it
  double sum = 0.0;
  bool nan = false;
  auto step = [&](const float (&x)[kBcPer], int i0) {
    float m = max3_nan(x[0], x[1], x[2]), m2 = max3_nan(x[3], x[4], x[5]);
#pragma unroll
    for (int j = 6; j + 4 <= kBcPer; j += 4) { m = max3_nan(m, x[j], x[j + 1]); m2 = max3_nan(m2, x[j + 2], x[j + 3]); }
    m = max3_nan(m, m2, max3_nan(m2, x[kBcPer - 2], x[kBcPer - 1]));
    if (m != m) { nan = true; m = -INFINITY; }                 // the row counts for nothing
    m = key_to_float(__reduce_max_sync(0xffffffffu, float_to_key(m)));
    if (lane == 0) out[i0 / kBcChunk] = m;
    if (m > top) {
      // The sum is kept relative to a power of two, which moves no bit of a term (and to e^base for logits beyond 1e6).
      const float new_base = fabsf(m) < 1e6f ? 0.f : m, new_n = rintf((m - new_base) * 1.44269504f);
      if (sum != 0.0) sum *= new_base == 0.f && base == 0.f ? pow2(big_n - new_n) : exp_of(((double)base - new_base) + ((double)big_n - new_n) * 0.6931471805599453);
      top = m; base = new_base; big_n = new_n; floor_x = m - 80.f;
    }
    if (top == -INFINITY) return;
    // e^x / 2^big_n by Cody and Waite's reduction (Software Manual for the Elementary Functions, 1980): x log2 e = n + f with log2 e in two
    // pieces, n into the exponent by integer arithmetic, 2^f (f exact to 2^-26) by ex2; two at a time.
    if (base == 0.f) {
      const float magic = 12582912.f - big_n;
      const unsigned long long log2e = f32x2(1.44269504f, 1.44269504f), rest = f32x2(1.92596299e-8f, 1.92596299e-8f), magic2 = f32x2(magic, magic),
                               minus = f32x2(-1.f, -1.f);
      unsigned long long a = 0ull, b = 0ull;
#pragma unroll
      for (int j = 0; j < kBcPer; j += 2) {
        // e^-80 of the largest is nothing in the sum's 53 bits, and -inf may count as that
        const unsigned long long y = f32x2(fmaxf(x[j], floor_x), fmaxf(x[j + 1], floor_x));
        const unsigned long long r = fma_f32x2(y, log2e, magic2), n = fma_f32x2(r, minus, magic2);
        float f0, f1, r0, r1;
        f32x2_split(fma_f32x2(y, rest, fma_f32x2(y, log2e, n)), f0, f1);
        f32x2_split(r, r0, r1);
        const unsigned long long e = f32x2(__int_as_float(__float_as_int(ex2_approx(f0)) + (__float_as_int(r0) << 23)),
                                           __int_as_float(__float_as_int(ex2_approx(f1)) + (__float_as_int(r1) << 23)));
        if (j & 2) b = add_f32x2(b, e); else a = add_f32x2(a, e);
      }
      float s0, s1;
      f32x2_split(add_f32x2(a, b), s0, s1);
      sum += (double)(s0 + s1);
    } else {                                                // big_n is 0
      float a = 0.f;
#pragma unroll
      for (int j = 0; j < kBcPer; ++j) a += x[j] >= floor_x ? expf(x[j] - base) : 0.f;
      sum += (double)a;
    }
  };
  int i = v0 + warp * kBcChunk;
  if (live && i < v1) {
    float x[kBcPer], y[kBcPer];
    load_chunk(x_row, i, v1, x);
    for (;;) {
      if (i + kBcTile < v1) load_chunk(x_row, i + kBcTile, v1, y);
      step(x, i);
      i += kBcTile;
      if (i >= v1) break;
      if (i + kBcTile < v1) load_chunk(x_row, i + kBcTile, v1, x);
      step(y, i);
      i += kBcTile;
      if (i >= v1) break;
    }
  }
  if (__any_sync(0xffffffffu, nan) || top == INFINITY) sum = __longlong_as_double(0x7ff8000000000000ll);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_part[warp] = {sum, (int)big_n, base};
  __syncthreads();
  if (warp == 0) {
    BeamPart p = s_part[lane % kBcWarps];
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
// at: beam * vocab + token (or a chunk's first token); key 0: none.  Equals go to the lower beam; within a beam, whose scores may be equal
// although its logits are not, to the larger logit, and then to the lower token.
struct BeamScore { unsigned long long key; int32_t at; uint32_t logit; };
constexpr BeamScore kNoScore = {0ull, 0x7fffffff, 0u};
__device__ __noinline__ bool equal_before(int a_at, uint32_t a_logit, int b_at, uint32_t b_logit, int vocab) {
  return a_at / vocab == b_at / vocab ? a_logit > b_logit : a_at < b_at;
}
struct BeamOrder {
  int vocab;
  __device__ __forceinline__ bool operator()(const BeamScore& a, const BeamScore& b) const {
    if (a.key != b.key) return a.key > b.key;
    return a.logit == b.logit ? a.at < b.at : equal_before(a.at, a.logit, b.at, b.logit, vocab);
  }
};
struct BeamQuestion {
  double lse[kBeamMax], score[kBeamMax];
  float least[kBeamMax];                                       // logits below it do not reach the bound
  unsigned long long key[kBjCap];                              // entries that wait to be ranked: BeamScore, its parts side by side
  int32_t at[kBjCap];
  uint32_t logit[kBjCap];
  BeamScore best[kBeamMaxK], one[kBjWarps];
  uint32_t post[kBjWarps];
  int count;
  __device__ __forceinline__ BeamScore of(float x, int b, int at) const {
    if (!(x > -INFINITY)) return kNoScore;
    x += 0.f;                                                  // -0 is 0
    const double v = score[b] + ((double)x - lse[b]);
    return v > -INFINITY && v < INFINITY ? BeamScore{score_key(v), at, float_to_key(x)} : kNoScore;
  }
  // 64-bit scores are for the few logits that may count: the others stay below a logit that gives less than `v`.  1e-12 of the
  // numbers involved is far more than those scores' own rounding.
  __device__ __forceinline__ void reach(double v, int b) {
    const double x = v - score[b] + lse[b];
    least[b] = __double2float_rd(x - 1e-12 * (fabs(v) + fabs(score[b]) + fabs(lse[b])));
  }
};

// The k best of what `each` hands to its argument, in order, into s.best; their number.
template <typename Each>
__device__ __forceinline__ int k_best(BeamQuestion& s, const BeamOrder& better, int k, const Each& each) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) s.count = 0;
  __syncthreads();
  each([&](const BeamScore& v) {
    const int i = atomicAdd(&s.count, 1);
    if (i < kBjCap) { s.key[i] = v.key; s.at[i] = v.at; s.logit[i] = v.logit; }
  });
  __syncthreads();
  int have = s.count;
  if (have > kBjCap) {                                        // equal scores, or chunks in order, by the hundred: one at a time
    BeamScore last{~0ull, -1, ~0u};
    for (have = 0; have < k; ++have) {
      BeamScore mine = kNoScore;
      each([&](const BeamScore& v) { if (better(last, v) && better(v, mine)) mine = v; });
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const BeamScore w = {__shfl_xor_sync(0xffffffffu, mine.key, o), __shfl_xor_sync(0xffffffffu, mine.at, o), __shfl_xor_sync(0xffffffffu, mine.logit, o)};
        if (better(w, mine)) mine = w;
      }
      if (lane == 0) s.one[warp] = mine;
      __syncthreads();
      mine = s.one[0];
      for (int w = 1; w < kBjWarps; ++w) if (better(s.one[w], mine)) mine = s.one[w];
      __syncthreads();
      if (!mine.key) break;
      if (tid == 0) s.best[have] = mine;
      last = mine;
    }
  } else {
    // Each entry's place is the number of better ones; four lanes count for an entry.
    for (int i = tid / 4; i < (have + 7) / 8 * 8; i += kBjThreads / 4) {
      const unsigned long long mine = i < have ? s.key[i] : 0ull;
      int place = 0, equal = 0;
#pragma unroll 4
      for (int o = tid % 4; o < have; o += 4) {
        const unsigned long long other = s.key[o];
        place += other > mine;
        equal += other == mine;
      }
      if (equal > (i % 4 == tid % 4)) {                        // besides itself
        const BeamScore v = {mine, s.at[i], s.logit[i]};
        for (int o = tid % 4; o < have; o += 4) if (s.key[o] == mine) place += better(BeamScore{mine, s.at[o], s.logit[o]}, v);
      }
      place += __shfl_xor_sync(0xffffffffu, place, 1);
      place += __shfl_xor_sync(0xffffffffu, place, 2);
      if (i < have && tid % 4 == 0 && place < k) s.best[place] = {mine, s.at[i], s.logit[i]};
    }
    have = min(have, k);
  }
  __syncthreads();
  return have;
}

struct BeamChoiceOut { float* score; int32_t *beam, *token; float* live_score; int32_t *live_beam, *live_token; };

// One block per question: the rows' sums, the k best chunks by their largest logits, and the k best of what lies in those.
template <typename T>
__global__ void __launch_bounds__(kBjThreads)
beam_join_kernel(const BeamPart* parts, const float* largest, const T* logits, long long stride, const float* scores, int beams, int vocab, int chunks,
                 int splits, int k, const int32_t* stop, int n_stop, const BeamChoiceOut out) {
  grid_dependency_wait();
  __shared__ BeamQuestion s;
  __shared__ BeamPart s_part[kBeamMax];
  __shared__ BeamScore s_chunk[kBeamMaxK];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long q = blockIdx.x;
  const BeamOrder better{vocab};
  // The chunks are dealt to the warps one by one, so that every warp sees some of every beam; a thread's first few are fetched here.
  const int n = beams * chunks, c0 = lane * kBjWarps + warp;
  float hold[kBjHold];
#pragma unroll
  for (int i = 0; i < kBjHold; ++i) hold[i] = i * kBjThreads + c0 < n ? largest[q * n + i * kBjThreads + c0] : -INFINITY;
  for (int b = warp; b < beams; b += kBjWarps) {
    BeamPart p = {0.0, 0, 0.f};
    for (int i = lane; i < splits; i += 32) join_sums(p, parts[(q * beams + b) * splits + i]);
    for (int o = 1; o < 32 && o < splits; o <<= 1) join_sums(p, other_part(p, o));
    if (lane == 0) s_part[b] = p;
  }
  __syncthreads();
  if (tid < beams) {                                          // nothing summed, or NaN: no candidates below
    const BeamPart p = s_part[tid];
    s.lse[tid] = ((double)p.base + (double)p.n * 0.6931471805599453) + log(p.sum);
    s.score[tid] = p.sum > 0.0 ? (double)scores[q * beams + tid] : -INFINITY;
    s.least[tid] = p.sum > 0.0 ? (float)(s.score[tid] - s.lse[tid]) : -INFINITY;        // what turns logits into scores, for now
  }
  __syncthreads();
  const float per_chunk = 1.f / (float)chunks;
  auto beam_of = [&](int c) {
    const int b = (int)(((float)c + 0.5f) * per_chunk);
    return c < b * chunks ? b - 1 : c >= (b + 1) * chunks ? b + 1 : b;
  };
  // A bound from below: every warp's `deep`-th best thread by the best of its chunks, and the `wide`-th best of the warps; in 32 bits, less
  // more than their rounding (two roundings of numbers no larger than these, 2^-24 each).  It lets some 1.5 k chunks pass.
  float top = -INFINITY, size = 0.f;
  auto see = [&](float x, int c) {
    const float off = s.least[beam_of(c)], v = x + off;
    if (v > top) { top = v; size = fabsf(off) + fabsf(v); }
  };
#pragma unroll
  for (int i = 0; i < kBjHold; ++i) if (i * kBjThreads + c0 < n) see(hold[i], i * kBjThreads + c0);
  for (int c = kBjHold * kBjThreads + c0; c < n; c += kBjThreads) see(largest[q * n + c], c);
  top -= size * 2.4e-7f;
  uint32_t key = top > -INFINITY && top < INFINITY ? float_to_key(top) : 0u, post = 0u;
  const int warps = min(kBjWarps, n), most = max(1, warps * 13 / 16), deep = (k + most - 1) / most, wide = (k + deep - 1) / deep;
  for (int i = 0; i < deep; ++i) {
    post = __reduce_max_sync(0xffffffffu, key);
    const unsigned who = __ballot_sync(0xffffffffu, key == post);
    if (lane == __ffs(who) - 1) key = 0u;
  }
  if (lane == 0) s.post[warp] = post;
  __syncthreads();
  if (warp == 0) {
    const uint32_t my_post = s.post[lane % kBjWarps];
    int place = 0;
    for (int w = 0; w < kBjWarps; ++w) place += s.post[w] > my_post || (s.post[w] == my_post && w < lane);
    const uint32_t bound = __shfl_sync(0xffffffffu, my_post, __ffs(__ballot_sync(0xffffffffu, lane < kBjWarps && place == wide - 1)) - 1);
    if (tid < beams) {
      if (bound) s.reach((double)key_to_float(bound), tid); else s.least[tid] = -INFINITY;
      if (!(s.score[tid] > -INFINITY)) s.least[tid] = INFINITY;
    }
  }
  __syncthreads();
  auto take = [&](float x, int c, auto&& use) {
    const int b = beam_of(c);
    if (x >= s.least[b] && x < INFINITY) {
      const BeamScore v = s.of(x, b, b * vocab + (c - b * chunks) * kBcChunk);
      if (v.key) use(v);
    }
  };
  const int picked = k_best(s, better, k, [&](auto&& use) {
#pragma unroll
    for (int i = 0; i < kBjHold; ++i) if (i * kBjThreads + c0 < n) take(hold[i], i * kBjThreads + c0, use);
    for (int c = kBjHold * kBjThreads + c0; c < n; c += kBjThreads) take(largest[q * n + c], c, use);
  });
  // The k-th chunk's largest is one of k logits that reach it.
  if (tid < picked) s_chunk[tid] = s.best[tid];
  if (tid < beams && picked == k) s.reach(key_score(s.best[k - 1].key), tid);
  __syncthreads();
  const int have = k_best(s, better, k, [&](auto&& use) {
    for (int c = warp; c < picked; c += kBjWarps) {
      const int b = s_chunk[c].at / vocab, i0 = s_chunk[c].at - b * vocab;
      const float least = s.least[b];
      const T* x_row = logits + (q * beams + b) * stride;
      float x[kBcPer];
      load_chunk(x_row, i0, vocab, x);
      uint32_t hits = 0u;
#pragma unroll
      for (int j = 0; j < kBcPer; ++j) hits |= x[j] >= least ? 1u << j : 0u;
      for (; hits; hits &= hits - 1u) {                        // few: read again rather than held in a register each
        const int i = i0 + (__ffs(hits) - 1) * 32 + lane;
        const BeamScore v = s.of(i < vocab ? to_f(x_row[i]) : -INFINITY, b, b * vocab + i);
        if (v.key) use(v);
      }
    }
  });
  if (tid < k) {
    const BeamScore v = s.best[tid];
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
      const BeamScore v = on ? s.best[c] : BeamScore{0ull, 0, 0u};
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
int launch_beam_topk(const void* logits, int64_t stride, const float* scores, int batch, int beams, int vocab, int chunks, int splits, int tiles_per_split, int k,
                     const int32_t* stop, int n_stop, BeamPart* parts, float* largest, const BeamChoiceOut& out, cudaStream_t st) {
  beam_rows_kernel<T><<<(unsigned)((int64_t)batch * beams * splits), kBcThreads, 0, st>>>((const T*)logits, stride, scores, vocab, chunks, splits,
                                                                                         tiles_per_split, parts, largest);
  MSA_LAUNCH_OK("beam_rows_kernel");
  MSA_CUDA_OK(launch_kernel_pdl(beam_join_kernel<T>, dim3((unsigned)batch), dim3(kBjThreads), 0, st, true, parts, largest, (const T*)logits, stride, scores, beams,
                                vocab, chunks, splits, k, stop, n_stop, out));
  MSA_LAUNCH_OK("beam_join_kernel");
  return MSA_OK;
}

}  // namespace msa

using namespace msa;

// Parts of a row, each of whole tiles: as many as let the blocks (kBcBlocks an SM at once) walk the fewest tiles one after the other, with one
// more tile's time for a block's start and end.
static int beam_splits(int64_t rows, int32_t vocab, int* tiles_per_split) {
  const int tiles = (vocab + kBcTile - 1) / kBcTile;
  int64_t best = 0;
  int per = tiles;
  for (int p = tiles; p >= 1; --p) {
    const int64_t blocks = rows * ((tiles + p - 1) / p), cost = (blocks + kBcBlocks * 148 - 1) / (kBcBlocks * 148) * (p + 1);
    if (best == 0 || cost < best) { best = cost; per = p; }
  }
  *tiles_per_split = per;
  return (tiles + per - 1) / per;
}

extern "C" int64_t msa_lm_beam_topk_workspace(int32_t batch, int32_t beams, int32_t vocab, int32_t k) {
  if (batch <= 0 || beams <= 0 || vocab <= 0 || k <= 0) return 0;
  int per = 0;
  const int64_t parts = (int64_t)batch * beams * beam_splits((int64_t)batch * beams, vocab, &per);
  return parts * (int64_t)sizeof(BeamPart) + (int64_t)batch * beams * ((vocab + kBcChunk - 1) / kBcChunk) * 4;
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
  float* largest = (float*)(parts + rows * splits);
  const BeamChoiceOut out{score, beam, token, live_score, live_beam, live_token};
  MSA_LM_DISPATCH(dtype, {
    return launch_beam_topk<T>(logits, stride, scores, batch, beams, vocab, (vocab + kBcChunk - 1) / kBcChunk, splits, per, k, stop, n_stop, parts, largest, out,
                               (cudaStream_t)stream);
  });
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
