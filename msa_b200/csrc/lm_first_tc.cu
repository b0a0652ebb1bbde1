// Attention of a prompt portion over a window with first tokens that stay visible, on the 5th-generation tensor cores (tcgen05 +
// TMEM + TMA), bf16, heads and values 64 or 128 wide.
//
//     o_i = g_i * sum_j p_ij v_j / (sink + sum_j p_ij),   p_ij = exp(s q_i . k_j),   j <= i and (i - j < window or j < first)
//
// Work item = 256 rows, two tiles of 128 that share every key / value tile on its way through shared memory.  A row is a token and
// one of 2^pack heads of a key head (as many as the group has factors of two, up to 32): a tile then spans fewer tokens, and fewer
// keys lie outside a row's window.  One persistent CTA per SM, 384 threads: warps 0-3 the softmax of tile 0, 4-7 that of tile 1 (thread =
// row = TMEM lane), warp 8 the TMA producer, warp 9 the MMA issuer, warp 10 finds the items, warp 11 clears values that are not the sequence's own.  Per 128 keys and row tile:
//     S = Q K^T    fp32 into the tile's 128 TMEM columns;
//     softmax      fp32; the reference moves only when the maximum is 2^32 above it (fp32 sums and bf16 weights keep their relative
//                  precision up to there, and O is rescaled all but never); P as bf16 over the consumed columns;
//     O += P V     A = P from TMEM, B = V MN-major; O stays in TMEM.
// While one tile's softmax runs, the tensor pipe works for the other.  128 keys because an issued product takes some 70 cycles
// whatever its columns: with 64 the issuing thread was the bound (3460 cycles for 64 keys of both tiles, 2200 of them issuing).  That
// thread is kept to one wait for copies, two for P and three commits per 128 keys: each costs it 90 to 140 cycles (4130 cycles an
// iteration with six of each).  Two issuing threads are slower (368 us where one took 298).
//
// Figures here are launches back to back of 4 portions of 2048 tokens, 32 heads over 8 of 128, window 2048, first and second of each pair on the same
// card, some before later steps and on other cards; as it stands the kernel takes 250 us so.
//
// Keys come as slots: the context's first rows up to a multiple of 8, then its rows from `base` on, the first that the item's window
// reaches (or where those rows end).  A tile in which the two meet is fetched by two copies, so that few first tokens cost no tile.
#include "lm_common.cuh"
#include "tc_attn_common.cuh"

namespace msa {

constexpr int kFtRows = 128, kFtTiles = 2, kFtKeys = 128;
constexpr int kFtThreads = 32 * (4 * kFtTiles + 4);
constexpr int kFtRing = 4;                                // items known ahead
constexpr int kFtBlk = kFtRows * 128;                     // one 64-column block of a row, key or value tile: 16 KB
constexpr int kFtKeyBufs = 3;
constexpr uint32_t kFtTmem = 512, kFtColO = kFtTiles * kFtKeys;
constexpr float kFtRescale = 32.f;

struct FirstAttnParams {
  const int32_t *start, *cu, *ctx_off;   // ctx_off counts from seq0
  int seq0, heads, window, first;
  int pad;                               // slots of the first rows
  int pack;                              // log2 of the heads that share a tile
  int q_row0;                            // packed row of the first query row of the map
  int k_head, v_head, group;             // column strides of a key / value head; query heads per key head
  int sink;                              // one more entry per softmax, with score 0 and no value
  const __nv_bfloat16* gate; long long gate_row;   // null, or one logit per row and head
  float scale_log2e;
  long long n_sh, n_items;               // sequences * head packs; times the blocks of the longest portion
  __nv_bfloat16* out; long long out_row;
  int32_t* status;
};

// Items are numbered from every portion's last block to its first: the late ones see the most keys, and the fixed-stride walk of the
// persistent CTAs then ends on short ones.  Row tile q takes part in the key tiles below f[q] and in a[q] .. b[q]-1.
struct FtItem {
  int len, tok0, h, q_row, ctx, old, shift, own, n_kt, f[kFtTiles], a[kFtTiles], b[kFtTiles];   // own: slots in front of the context's end
  uint32_t turn;                                             // turns of the items before it
  bool valid;
  __device__ __forceinline__ bool foreign() const { return own < n_kt * kFtKeys; }       // rows in the last key tile
  __device__ __forceinline__ bool has(int q, int t) const { return t < f[q] || (t >= a[q] && t < b[q]); }
};
__device__ __forceinline__ FtItem ft_item(const FirstAttnParams& p, long long w) {
  FtItem it;
  const uint32_t n_sh = (uint32_t)p.n_sh;
  const int x = (int)((uint32_t)w / n_sh), packs = p.heads >> p.pack, span = (kFtRows * kFtTiles) >> p.pack, each = kFtRows >> p.pack;
  const int sh = (int)((uint32_t)w - (uint32_t)x * n_sh), ps = sh / packs, s = p.seq0 + ps;
  it.h = (sh - ps * packs) << p.pack;
  const int c0 = p.cu[s];
  it.len = p.cu[s + 1] - c0;
  const int n_mb = (it.len + span - 1) / span;
  it.valid = x < n_mb;
  it.tok0 = (n_mb - 1 - x) * span;
  it.old = old_rows(p.start[s], p.first + p.window);
  it.q_row = c0 - p.q_row0 + it.tok0;
  it.ctx = p.ctx_off[ps];
  it.shift = max(p.pad, it.old + it.tok0 - p.window + 1) - p.pad;      // context row = slot + shift behind the first rows
  it.own = it.old + it.len - it.shift;
  it.n_kt = 0;
#pragma unroll
  for (int q = 0; q < kFtTiles; ++q) {
    const int t0 = it.tok0 + q * each, t1 = min(t0 + each, it.len);
    it.f[q] = it.a[q] = it.b[q] = 0;
    if (t0 < it.len) {
      const int end = it.old + t1 - it.shift;                          // behind the last row's own key, as a slot
      it.f[q] = (min(p.pad, end) + kFtKeys - 1) / kFtKeys;
      it.a[q] = max(p.pad, it.old + t0 - p.window + 1 - it.shift) / kFtKeys;
      it.b[q] = (end + kFtKeys - 1) / kFtKeys;
      it.n_kt = max(it.n_kt, it.b[q]);
    }
  }
  return it;
}

// Slots (lo, hi] of the 32 from s0 on, as bits.
__device__ __forceinline__ uint32_t slot_bits(int lo, int hi, int s0) {
  const int l = min(max(lo - s0 + 1, 0), 32), h = min(max(hi - s0 + 1, 0), 32);
  const uint32_t below_h = h == 32 ? ~0u : (1u << h) - 1u, below_l = l == 32 ? ~0u : (1u << l) - 1u;
  return below_h & ~below_l;
}

__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
// A store that leaves no line in the L1, which shared memory holds nearly all of: 5 us of 262.
__device__ __forceinline__ void store_once(void* p, uint4 v) {
  asm volatile("st.global.L1::no_allocate.v4.b32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

template <int DB, int VB>
__global__ void __launch_bounds__(kFtThreads, 1)
first_attn_tc_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_k0,
                     const __grid_constant__ CUtensorMap tmap_k1, const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ CUtensorMap tmap_v0,
                     const __grid_constant__ CUtensorMap tmap_v1, const FirstAttnParams p) {
  static_assert(kFtColO + kFtTiles * VB * 64 <= kFtTmem, "TMEM columns");
  extern __shared__ unsigned char smem_dyn[];
  __shared__ uint64_t s_q_full, s_q_empty, s_kv_full[2], s_kv_empty[2], s_dirty, s_clean, s_drain;
  __shared__ uint64_t s_s_full[kFtTiles], s_p_full[kFtTiles], s_o_full[kFtTiles];
  __shared__ uint32_t s_tmem_base;
  __shared__ int s_abort;
  __shared__ FtItem s_item[kFtRing];
  __shared__ uint64_t s_item_full[kFtRing], s_item_empty[kFtRing];

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  unsigned char* tiles = reinterpret_cast<unsigned char*>(((uintptr_t)smem_dyn + 1023) & ~(uintptr_t)1023);
  unsigned char* q_smem = tiles;
  unsigned char* k_smem = q_smem + kFtTiles * DB * kFtBlk;
  unsigned char* v_smem = k_smem + kFtKeyBufs * DB * kFtBlk;
  volatile int* abort_flag = &s_abort;

  if (threadIdx.x == 0) {
    mbar_init(&s_q_full, 1); mbar_init(&s_q_empty, 1); mbar_init(&s_dirty, 1); mbar_init(&s_clean, 1); mbar_init(&s_drain, 1);
    for (int i = 0; i < 2; ++i) { mbar_init(&s_kv_full[i], 1); mbar_init(&s_kv_empty[i], 1); }
    for (int q = 0; q < kFtTiles; ++q) {
      mbar_init(&s_s_full[q], 1); mbar_init(&s_p_full[q], 4); mbar_init(&s_o_full[q], 1);
    }
    for (int i = 0; i < kFtRing; ++i) { mbar_init(&s_item_full[i], 1); mbar_init(&s_item_empty[i], 4 * kFtTiles + 3); }
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 4 * kFtTiles + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem_base)),
                 "r"(kFtTmem) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = s_tmem_base;

  // Every role walks the same items, which warp 10 puts into a ring: found by the roles themselves, each item began with 1500 to 3500 cycles
  // of loads behind the last one's stores.  Keys come one tile ahead of their values: an item starts with its queries and first keys, and turn t
  // brings the values of tile t with the keys of tile t + 1.  n_t counts the turns (stage and phase of the K / V barriers), n_c the tiles
  // that a row tile took part in (phase of its S and P barriers), n_o its items, n_it all items.  Turn n_t waits for the end of turn n_t - 2,
  // in front of which S of an item's first keys may not have been issued: three buffers of keys, taken in turn (b_k), so that
  // those are overwritten two turns after S's own.
  auto item_wait = [&](uint32_t n) { return mbar_wait(&s_item_full[n % kFtRing], (n / kFtRing) & 1u, abort_flag, p.status, 7); };
  if (warp == 4 * kFtTiles + 2) {
    if (lane == 0) {
      uint32_t n = 0, turn = 0;
      for (long long w = blockIdx.x;; w += gridDim.x) {
        FtItem it{};                                          // behind the last one: not valid, which ends the walk
        if (w < p.n_items) {
          it = ft_item(p, w);
          if (!it.valid) continue;
        }
        if (!mbar_wait(&s_item_empty[n % kFtRing], ((n / kFtRing) & 1u) ^ 1u, abort_flag, p.status, 7)) break;
        it.turn = turn;
        turn += (uint32_t)it.n_kt;
        s_item[n % kFtRing] = it;
        mbar_arrive(&s_item_full[n % kFtRing]);
        ++n;
        if (w >= p.n_items) break;
      }
    }
  } else if (warp == 4 * kFtTiles + 3) {
    // Rows behind the portion's context belong to another sequence, or to nobody.  Their weights are 0, which would still take an infinity or
    // a NaN from their values into the product: they are cleared before it.  (By the softmax warps, this cost all tiles 15 us of 265.)
    bool ok = true;
    uint32_t n_cl = 0;
    for (uint32_t n_it = 0; ok; ++n_it) {
      ok = __all_sync(0xffffffffu, item_wait(n_it));
      if (!ok) break;
      const FtItem& it = s_item[n_it % kFtRing];
      const bool more = it.valid, foreign = it.foreign();
      const int own = it.own - (it.n_kt - 1) * kFtKeys;
      const uint32_t n = it.turn + (uint32_t)it.n_kt - 1u;
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_item_empty[n_it % kFtRing]);
      if (!more) break;
      if (!foreign) continue;
      ok = __all_sync(0xffffffffu, mbar_wait(&s_dirty, n_cl++ & 1u, abort_flag, p.status, 8));      // the tile has come
      if (!ok) break;
      for (int i = own * 8 + lane; i < kFtKeys * 8; i += 32)
#pragma unroll
        for (int c = 0; c < VB; ++c) *reinterpret_cast<uint4*>(v_smem + ((n & 1u) * VB + c) * kFtBlk + i * 16) = make_uint4(0u, 0u, 0u, 0u);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_clean);
    }
  } else if (warp == 4 * kFtTiles) {
    if (lane == 0) {
      uint32_t n_it = 0, n_t = 0, b_k = 0;
      bool ok = true;
      auto next = [](uint32_t b) { return b + 1 == kFtKeyBufs ? 0u : b + 1; };
      // One key or value tile: slots 128 t .. of `heads` columns from x on.
      auto load = [&](unsigned char* dst, const CUtensorMap* full, const CUtensorMap* front, const CUtensorMap* back, int blocks, int x, const FtItem& it, int t,
                      uint64_t* bar) {
        const int s0 = t * kFtKeys, n_front = p.pad - s0;       // slots of this tile that are first rows
        for (int c = 0; c < blocks; ++c) {
          unsigned char* d = dst + c * kFtBlk;
          if (n_front > 0 && n_front < kFtKeys) {
            tma_load_2d(d, front, x + 64 * c, it.ctx + s0, bar);
            tma_load_2d(d + n_front * 128, back, x + 64 * c, it.ctx + p.pad + it.shift, bar);
          } else {
            tma_load_2d(d, full, x + 64 * c, it.ctx + s0 + (n_front > 0 ? 0 : it.shift), bar);
          }
        }
      };
      while (ok && (ok = item_wait(n_it))) {
        const FtItem it = s_item[n_it % kFtRing];
        mbar_arrive(&s_item_empty[n_it % kFtRing]);
        if (!it.valid) break;
        if (!(ok = mbar_wait(&s_q_empty, (n_it & 1u) ^ 1u, abort_flag, p.status, 1))) break;
        const int k_col = it.h / p.group * p.k_head, v_col = it.h / p.group * p.v_head;
        mbar_expect_tx(&s_q_full, (kFtTiles + 1) * DB * kFtBlk);
#pragma unroll
        for (int q = 0; q < kFtTiles; ++q)
#pragma unroll
          for (int c = 0; c < DB; ++c)
            tma_load_3d(q_smem + (q * DB + c) * kFtBlk, &tmap_q, 64 * c, it.h, it.q_row + q * (kFtRows >> p.pack), &s_q_full);
        load(k_smem + b_k * DB * kFtBlk, &tmap_k, &tmap_k0, &tmap_k1, DB, k_col, it, 0, &s_q_full);
        b_k = next(b_k);
        for (int t = 0; t < it.n_kt; ++t, ++n_t) {
          const uint32_t st = n_t & 1u, ph = (n_t >> 1) & 1u;
          const bool more = t + 1 < it.n_kt;
          if (!(ok = mbar_wait(&s_kv_empty[st], ph ^ 1u, abort_flag, p.status, 1))) break;
          mbar_expect_tx(&s_kv_full[st], (VB + (more ? DB : 0)) * kFtBlk);
          load(v_smem + st * VB * kFtBlk, &tmap_v, &tmap_v0, &tmap_v1, VB, v_col, it, t, &s_kv_full[st]);
          if (more) {
            load(k_smem + b_k * DB * kFtBlk, &tmap_k, &tmap_k0, &tmap_k1, DB, k_col, it, t + 1, &s_kv_full[st]);
            b_k = next(b_k);
          }
        }
        ++n_it;
      }
      if (!ok) {   // gave up: give the copies already issued time to land before shared memory is released
        const unsigned long long w0 = global_ns();
        while (global_ns() - w0 < 1000000ull) {}
      }
    }
  } else if (warp == 4 * kFtTiles + 1) {
    // The whole warp walks along, and one thread (always the same) issues: with the others left behind at a branch around all of this, each
    // product's descriptors cost more than the product (261 us against 256).
    const uint32_t idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(kFtKeys >> 3) << 17) | ((uint32_t)(kFtRows >> 4) << 24);
    const uint32_t idesc_pv = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(VB * 64 >> 3) << 17) |
                              ((uint32_t)(kFtRows >> 4) << 24);
    const uint64_t q_desc = make_smem_desc(smem_u32(q_smem)), k_desc = make_smem_desc(smem_u32(k_smem)),
                   v_desc = make_smem_desc_mn(smem_u32(v_smem), kFtBlk);
    uint32_t n_it = 0, n_t = 0, n_cl = 0, b_k = 0, n_p[kFtTiles] = {};   // n_cl: tiles that were cleared, n_p: PV tiles issued so far
    bool ok = true;
    auto all_wait = [&](uint64_t* bar, uint32_t ph, int code) { return (bool)__all_sync(0xffffffffu, mbar_wait(bar, ph, abort_flag, p.status, code)); };
    auto issue_s = [&](uint32_t g, int q) {                // S of the keys in buffer g for row tile q
      if (!elect_one()) return;
      const uint64_t b_desc = k_desc + (uint64_t)(g * (DB * kFtBlk >> 4));
#pragma unroll
      for (int c = 0; c < DB; ++c)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          tc_mma_bf16(tmem_base + (uint32_t)(q * kFtKeys), q_desc + (uint64_t)(((q * DB + c) * kFtBlk >> 4) + 2 * k),
                      b_desc + (uint64_t)((c * kFtBlk >> 4) + 2 * k), idesc_s, (c > 0 || k > 0) ? 1u : 0u);
      tc_commit(&s_s_full[q]);
    };
    while (ok && (ok = __all_sync(0xffffffffu, item_wait(n_it)))) {
      const FtItem it = s_item[n_it % kFtRing];
      __syncwarp();
      if (elect_one()) mbar_arrive(&s_item_empty[n_it % kFtRing]);
      if (!it.valid) break;
      if (!(ok = all_wait(&s_q_full, n_it & 1u, 2))) break;
      tc_fence_after();
#pragma unroll
      for (int q = 0; q < kFtTiles; ++q)
        if (it.has(q, 0)) issue_s(b_k, q);                  // behind the last item's products that read these columns
      b_k = b_k + 1 == kFtKeyBufs ? 0u : b_k + 1;
      if (it.n_kt == 1 && elect_one()) tc_commit(&s_q_empty);
      for (int t = 0; t < it.n_kt; ++t, ++n_t) {
        const uint32_t st = n_t & 1u;
        const bool more = t + 1 < it.n_kt;
        if (!(ok = all_wait(&s_kv_full[st], (n_t >> 1) & 1u, 3))) break;
        if (!more && it.foreign()) {
          if (elect_one()) mbar_arrive(&s_dirty);
          if (!(ok = all_wait(&s_clean, n_cl++ & 1u, 8))) break;
        }
        const uint64_t b_desc = v_desc + (uint64_t)(st * (VB * kFtBlk >> 4));
#pragma unroll
        for (int q = 0; q < kFtTiles; ++q) {
          if (it.has(q, t)) {
            if (!(ok = all_wait(&s_p_full[q], n_p[q] & 1u, 4))) break;
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int j = 0; j < kFtKeys / 16; ++j)
                tc_mma_bf16_ts(tmem_base + kFtColO + (uint32_t)(q * VB * 64), tmem_base + (uint32_t)(q * kFtKeys + 8 * j), b_desc + (uint64_t)(j * (2048 >> 4)),
                               idesc_pv, t > 0 || j > 0 ? 1u : 0u);
              if (t + 1 == it.b[q]) tc_commit(&s_o_full[q]);
            }
            ++n_p[q];
          }
          if (more && it.has(q, t + 1)) issue_s(b_k, q);    // in order behind the PV that read these columns
        }
        if (!ok) break;
        if (more) b_k = b_k + 1 == kFtKeyBufs ? 0u : b_k + 1;
        if (elect_one()) {
          tc_commit(&s_kv_empty[st]);
          if (t + 2 == it.n_kt) tc_commit(&s_q_empty);
        }
      }
      ++n_it;
    }
    if (elect_one()) tc_commit(&s_drain);
    const unsigned long long w0 = global_ns();
    while (!mbar_try_wait(&s_drain, 0) && global_ns() - w0 < kWaitLimitNs) {}
  } else {
    const int q = warp / 4, wq = warp % 4;
    const uint32_t lane_base = tmem_base + ((uint32_t)(wq * 32) << 16);
    const uint32_t s_addr = lane_base + (uint32_t)(q * kFtKeys), o_addr = lane_base + kFtColO + (uint32_t)(q * VB * 64);
    uint32_t n_c = 0, n_o = 0;
    bool ok = true;
    for (uint32_t n_it = 0; ok; ++n_it) {
      ok = item_wait(n_it);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const FtItem& it = s_item[n_it % kFtRing];              // kept until the item's end: registers are short
      if (!it.valid) break;
      const int f_q = it.f[q], a_q = it.a[q], b_q = it.b[q];
      auto release = [&] {
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_item_empty[n_it % kFtRing]);
      };
      const int t_first = it.tok0 + q * (kFtRows >> p.pack);
      if (t_first >= it.len) { release(); continue; }
      const int r_first = it.q_row - it.tok0 + t_first;       // row of the tile's first token in q and out
      const int low = (1 << p.pack) - 1, r_mine = wq * 32 + lane;
      // The gate is on its way during the tiles; a sigmoid of infinity is 1.
      const bool gated = p.gate && t_first + (r_mine >> p.pack) < it.len;
      unsigned short gate = 0x7f80;
      if (gated) gate = reinterpret_cast<const unsigned short*>(p.gate)[(long long)(r_first + (r_mine >> p.pack)) * p.gate_row + it.h + (r_mine & low)];
      float m_ref = p.sink ? 0.f : -1e30f, l_run = p.sink ? 1.f : 0.f;
      const int row0 = t_first + ((wq * 32) >> p.pack), row1 = t_first + ((wq * 32 + 31) >> p.pack);   // this warp's tokens
      const int mine = it.old + t_first + ((wq * 32 + lane) >> p.pack);                                // context row of the lane's token
      bool joined = false;                                    // O holds something of this item
      for (int t = 0; t < b_q; t = t + 1 < f_q || t + 1 >= a_q ? t + 1 : a_q) {
        ok = mbar_wait(&s_s_full[q], n_c & 1u, abort_flag, p.status, 5);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        uint32_t v[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(s_addr + 32 * c, v[c]);
        tmem_ld_wait();
        const int s_tile = t * kFtKeys, k_tile = s_tile + it.shift - it.old;       // first slot, and its token if none are first rows
        if (s_tile < p.pad || k_tile + kFtKeys - 1 > row0 || k_tile <= row1 - p.window) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int s0 = s_tile + 32 * c;
            uint32_t seen = slot_bits(mine - p.window - it.shift, mine - it.shift, s0);
            if (s0 < p.pad) {
              const uint32_t front = slot_bits(s0 - 1, p.pad - 1, s0);
              seen = (seen & ~front) | ((slot_bits(-1, min(p.first - 1, mine), s0) | slot_bits(mine - p.window, mine, s0)) & front);
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) if (!((seen >> i) & 1u)) v[c][i] = 0xff800000u;
          }
        }
        float mx[8];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          mx[2 * c] = __uint_as_float(v[c][0]);
          mx[2 * c + 1] = __uint_as_float(v[c][1]);
#pragma unroll
          for (int i = 2; i < 30; i += 4) {
            mx[2 * c] = max3(mx[2 * c], __uint_as_float(v[c][i]), __uint_as_float(v[c][i + 1]));
            mx[2 * c + 1] = max3(mx[2 * c + 1], __uint_as_float(v[c][i + 2]), __uint_as_float(v[c][i + 3]));
          }
          mx[2 * c] = max3(mx[2 * c], __uint_as_float(v[c][30]), __uint_as_float(v[c][31]));
        }
        const float top = max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], mx[4], mx[5]), fmaxf(mx[6], mx[7]));
        const bool move = (top - m_ref) * p.scale_log2e > kFtRescale;
        if (__any_sync(0xffffffffu, move)) {
          const float f = move ? exp2f((m_ref - top) * p.scale_log2e) : 1.f;
          if (joined) {        // S came behind the last PV: rescale this warp's rows of O in place
#pragma unroll
            for (int c = 0; c < VB * 4; ++c) {
              uint32_t o[16];
              tmem_ld16(o_addr + 16 * c, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              tmem_st16(o_addr + 16 * c, o);
            }
          }
          l_run *= f;
          if (move) m_ref = top;
        }
        const float neg_m = -m_ref * p.scale_log2e;
        unsigned long long sum_a = 0ull, sum_b = 0ull;
        const unsigned long long scale2 = f32x2(p.scale_log2e, p.scale_log2e), neg_m2 = f32x2(neg_m, neg_m);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            float x0, x1, x2, x3;
            f32x2_split(fma_f32x2(f32x2(__uint_as_float(v[c][i]), __uint_as_float(v[c][i + 1])), scale2, neg_m2), x0, x1);
            f32x2_split(fma_f32x2(f32x2(__uint_as_float(v[c][i + 2]), __uint_as_float(v[c][i + 3])), scale2, neg_m2), x2, x3);
            const float e0 = ex2_approx(x0), e1 = ex2_approx(x1), e2 = ex2_approx(x2), e3 = ex2_approx(x3);
            sum_a = add_f32x2(sum_a, f32x2(e0, e1));
            sum_b = add_f32x2(sum_b, f32x2(e2, e3));
            pk[i >> 1] = pack2_bf16(e0, e1);
            pk[(i >> 1) + 1] = pack2_bf16(e2, e3);
          }
          tmem_st16(s_addr + 16 * c, pk);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_p_full[q]);
        float s0, s1, s2, s3;
        f32x2_split(sum_a, s0, s1);
        f32x2_split(sum_b, s2, s3);
        l_run += (s0 + s1) + (s2 + s3);
        joined = true;
        ++n_c;
      }
      if (!ok) break;
      ok = mbar_wait(&s_o_full[q], n_o++ & 1u, abort_flag, p.status, 6);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const float inv = sigmoid_f(__uint_as_float((uint32_t)gate << 16)) / l_run;
      // Eight rows of 64 bytes a store: lanes trade the 16-byte pieces of their rows, the piece's two bits for the lane's upper two.
      const int hi = lane >> 4, mid = (lane >> 3) & 1, piece = lane >> 3;
      __nv_bfloat16* dst[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = wq * 32 + 8 * i + (lane & 7), tok = r >> p.pack;
        dst[i] = t_first + tok < it.len ? p.out + (long long)(r_first + tok) * p.out_row + (it.h + (r & low)) * VB * 64 + 8 * piece : nullptr;
      }
#pragma unroll 1                                              // run once an item: unrolled, it waits for its instructions
      for (int c = 0; c < VB * 2; ++c) {
        uint32_t o[32], d[16];                                // d: [piece][word]
        tmem_ld32(o_addr + 32 * c, o);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) d[i] = pack2_bf16(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
#pragma unroll
        for (int i = 0; i < 8; ++i) {                         // pieces 2, 3 of the lower lanes against 0, 1 of the upper ones
          const uint32_t got = __shfl_xor_sync(0xffffffffu, hi ? d[i] : d[8 + i], 16);
          if (hi) d[i] = got; else d[8 + i] = got;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int at = (i >> 2) * 8 + (i & 3);
          const uint32_t got = __shfl_xor_sync(0xffffffffu, mid ? d[at] : d[at + 4], 8);
          if (mid) d[at] = got; else d[at + 4] = got;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (dst[i]) store_once(dst[i] + 32 * c, make_uint4(d[4 * i], d[4 * i + 1], d[4 * i + 2], d[4 * i + 3]));
      }
      release();
      tc_fence_before();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 4 * kFtTiles + 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kFtTmem) : "memory");
}

template <int DB, int VB>
int launch_first_attn_tc(const CUtensorMap& q, const CUtensorMap (&k)[3], const CUtensorMap (&v)[3], const FirstAttnParams& p, cudaStream_t stream) {
  constexpr size_t smem = (size_t)((kFtTiles + kFtKeyBufs) * DB + 2 * VB) * kFtBlk + 1024;
  static_assert(smem <= 227 * 1024, "shared memory");
  static DeviceSmem configured{};
  MSA_OK_OR_RETURN(ensure_dynamic_smem(first_attn_tc_kernel<DB, VB>, smem, configured));
  int n_sm = 0;
  MSA_OK_OR_RETURN(device_sm_count(&n_sm));
  const long long grid = p.n_items < n_sm ? p.n_items : n_sm;
  first_attn_tc_kernel<DB, VB><<<(unsigned)grid, kFtThreads, smem, stream>>>(q, k[0], k[1], k[2], v[0], v[1], v[2], p);
  MSA_LAUNCH_OK("first_attn_tc_kernel");
  return MSA_OK;
}

// Keys or values [n_ctx, heads * head columns] in boxes of a whole tile, of the slots that are first rows in the tile where those end, and of
// the rest of that tile.
static int context_maps(CUtensorMap (&map)[3], const void* base, int64_t n_ctx, int64_t cols, int64_t row, int pad) {
  const int front = pad % kFtKeys;
  MSA_OK_OR_RETURN(make_map(&map[0], base, n_ctx, cols, row, 64, kFtKeys));
  map[1] = map[2] = map[0];
  if (front) {
    MSA_OK_OR_RETURN(make_map(&map[1], base, n_ctx, cols, row, 64, front));
    MSA_OK_OR_RETURN(make_map(&map[2], base, n_ctx, cols, row, 64, kFtKeys - front));
  }
  return MSA_OK;
}

}  // namespace msa

using namespace msa;

// The checks of arguments are msa_lm_window_attn_tc_first's.
int msa::first_attn_tc(const msa_lm_attn_args& a, int first, int n_rows, int n_ctx, int row0, int32_t* status, cudaStream_t stream) {
  const int kv_heads = a.heads / a.group;
  int pack = 0;
  while (pack < 5 && (a.group >> pack) % 2 == 0) ++pack;
  FirstAttnParams p{};
  p.start = a.start; p.cu = a.cu; p.ctx_off = a.ctx_off;
  p.seq0 = a.seq0; p.heads = a.heads; p.window = a.window; p.first = first; p.pad = (first + 7) / 8 * 8; p.pack = pack; p.q_row0 = row0;
  p.k_head = (int)a.ka_head; p.v_head = (int)a.v_head; p.group = a.group; p.sink = a.sink;
  p.gate = (const __nv_bfloat16*)a.gate; p.gate_row = a.gate_row;
  p.scale_log2e = a.scale * 1.4426950408889634f;
  const int span = (kFtRows * kFtTiles) >> pack;
  p.n_sh = (long long)(a.seq1 - a.seq0) * (a.heads >> pack);
  p.n_items = p.n_sh * ((a.max_len + span - 1) / span);
  MSA_REQUIRE(p.n_items < (1ll << 31), "window_attn_tc: too many rows");
  p.out = (__nv_bfloat16*)a.out; p.out_row = a.out_row; p.status = status;
  CUtensorMap mq, mk[3], mv[3];
  MSA_OK_OR_RETURN(make_map_heads(&mq, a.qa, n_rows, a.heads, a.da, a.qa_row, a.qa_head, 1u << pack, (uint32_t)kFtRows >> pack));
  MSA_OK_OR_RETURN(context_maps(mk, a.ka, n_ctx, (int64_t)(kv_heads - 1) * a.ka_head + a.da, a.ka_row, p.pad));
  MSA_OK_OR_RETURN(context_maps(mv, a.v, n_ctx, (int64_t)(kv_heads - 1) * a.v_head + a.dv, a.v_row, p.pad));
  if (a.da == 64) return a.dv == 64 ? launch_first_attn_tc<1, 1>(mq, mk, mv, p, stream) : launch_first_attn_tc<1, 2>(mq, mk, mv, p, stream);
  return a.dv == 64 ? launch_first_attn_tc<2, 1>(mq, mk, mv, p, stream) : launch_first_attn_tc<2, 2>(mq, mk, mv, p, stream);
}
