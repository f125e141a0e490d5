// Attention over a paged cache with all q-heads of a kv head in one tile of rows, on tcgen05 / TMEM.  Two users:
//   PREFILL  several tokens per sequence with a sliding window and sinks: the query at position p sees the keys j <= p
//            with j >= p - window or j < sinks; normalised output
//   PREFIX   one token per sequence, the sequences of a group against the prefix that they share: every row sees every
//            key, the keys cut into splits, unnormalised output + (maximum, sum) of every split, which
//            cluster_decode.cu joins with the sequences' own tokens
//
// Scores q.k * sm_scale (optional tanh soft-cap), softmax with a running maximum (raised only when it grew by 2^8) and sum
// in 32 bits, P rounded to the cache's 16-bit type for the second product (half a step of 2^-8 / 2^-11 on weights that
// are then averaged), accumulation in 32 bits.
//
// Row r of a tile is token r / group, q-head r % group of the kv head, so a tile of 128 rows is 128 / group tokens: a key
// tile is fetched once for all heads that share it, a window costs window + 128 / group keys instead of window + 128,
// five tokens of a sequence fill 20 to 35 rows of one tile instead of 5 rows of four to seven, and 256 sequences behind
// one prefix are 8 tiles of 128 rows with 4 heads each.  q arrives by one TMA box per 64 columns
// ([tokens, heads, columns] boxes land in that row order).
//
// One CTA = one (row tile, kv head, split), two CTAs per SM (256 TMEM columns and about 97 KiB each), so that one CTA's
// softmax runs beside the other's matrix instructions.  192 threads: warp 4 issues the loads (K and V tiles of 64 keys into
// 2-stage rings, one box per page), one lane of warp 5 the tcgen05.mma (S_j = Q K_j^T into one of two S buffers, then
// O += P_{j-1} V_{j-1} with P as the A operand from TMEM), warps 0-3 the softmax, one thread per row.  The blocks of
// 64 keys are those of the sinks and then those of the window; blocks in between are skipped, and so are pages
// that hold no key which the tile sees.
#include <math_constants.h>

#include "cluster_decode.cuh"

namespace dlb {

namespace pa {
constexpr int BM = 128;           // rows per CTA
constexpr int BN = 64;            // keys per block
constexpr int THREADS = 192;      // warps 0-3 softmax (TMEM quadrant = warp id), warp 4 TMA, warp 5 MMA
constexpr int WARP_TMA = 4;
constexpr int WARP_MMA = 5;
constexpr int Q_BOX = BM * 128;   // one 64-wide (128 B) column box of the Q tile
constexpr int KV_BOX = BN * 128;  // one 64-wide column box of a K or V tile
constexpr int KV_STAGES = 2;
constexpr int TMEM_COLS = 256;    // S0 [0,64) S1 [64,128) O [128,128+D)
constexpr float RESCALE_THRESHOLD = 8.0f;   // log2 units: P stays below 2^8, well inside fp16
enum { PREFILL, PREFIX };
template <int D> struct Layout {
  static constexpr int BOXES = D / 64;
  static constexpr int KV_BYTES = BOXES * KV_BOX;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = OFF_Q + BOXES * Q_BOX;
  static constexpr int OFF_V = OFF_K + KV_STAGES * KV_BYTES;
  static constexpr int OFF_CTRL = OFF_V + KV_STAGES * KV_BYTES;
  static constexpr int SMEM_BYTES = OFF_CTRL + 160;
};
}  // namespace pa

struct PackedParams {
  void* out;                      // PREFILL: [tokens, hq, dv]
  const void* q_start;            // PREFILL: [batch] first row of each sequence, its rows, its keys (new ones included)
  const void* q_lens;
  const void* kv_lens;
  const void* block_table;        // [batch, max_pages]; PREFIX: one row per group
  int64_t o_st, o_sh, bt_stride;
  int64_t tokens;                 // rows of q
  int batch;                      // sequences, or groups
  int hq, hkv, group, tile_tokens;
  uint32_t group_inv;             // ceil(2^16 / group): r / group = r * group_inv >> 16 for r < 128
  int tiles;                      // row tiles in the grid
  int page_shift, max_pages, num_pages, dv;
  int table_is_int64, start_is_int64, qlens_is_int64, lens_is_int64;
  int window, sinks;              // PREFILL
  float scale_log2, sm_scale, softcap;
  uint32_t idesc_qk, idesc_pv;
  int* status;
  PrefixPartials prefix;          // PREFIX
};

// Row tile x of the launch -> sequence (or group) and tile inside it, its rows and keys; false if there is none.  The tiles
// that exist are numbered through, sequence by sequence, 32 sequences at a time over the lanes of a warp (every warp does it
// for itself), so that a batch of any lengths needs no more CTAs than it has tiles.
template <int MODE>
__device__ __forceinline__ bool packed_tile(const PackedParams& p, int x, int& seq, int& tile, int& start, int& n, int& kv_len) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    const int b = b0 + lane;
    int st = 0, rows = 0, keys = 0;
    if (b < p.batch) {
      if (MODE == pa::PREFIX) {
        group_rows(p.prefix, p.tokens, b, st, rows);
        keys = load_index(p.prefix.lens, b, p.prefix.lens_is_int64);
      } else {
        // rows outside q are nobody's
        st = load_index(p.q_start, b, p.start_is_int64);
        rows = load_index(p.q_lens, b, p.qlens_is_int64);
        keys = load_index(p.kv_lens, b, p.lens_is_int64);
        rows = (st < 0 || st >= p.tokens) ? 0 : (int)min((int64_t)max(rows, 0), p.tokens - st);
      }
    }
    const int mine = (rows + p.tile_tokens - 1) / p.tile_tokens;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, before + upto > x);
    if (past != 0) {
      const int src = __ffs(past) - 1;
      seq = b0 + src;
      const int of_seq = __shfl_sync(0xffffffffu, mine, src);
      tile = of_seq - 1 - (x - (before + __shfl_sync(0xffffffffu, upto, src) - of_seq));   // the late, long ones first
      start = __shfl_sync(0xffffffffu, st, src);
      n = __shfl_sync(0xffffffffu, rows, src);
      kv_len = __shfl_sync(0xffffffffu, keys, src);
      return true;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return false;
}

template <typename T, int D, int MODE, bool CAP>
__global__ void __launch_bounds__(pa::THREADS, 2)
packed_attention_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                        const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ PackedParams p) {
  using namespace pa;
  using L = Layout<D>;
  constexpr int BOXES = L::BOXES, KV_BYTES = L::KV_BYTES;
  constexpr int OFF_Q = L::OFF_Q, OFF_K = L::OFF_K, OFF_V = L::OFF_V, OFF_CTRL = L::OFF_CTRL;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  // ---- which tile: PREFILL has the kv heads of a tile side by side, PREFIX the row tiles of a (kv head, split), which
  // read the same keys ----
  int x = (int)blockIdx.x, kvh, split = 0;
  if (MODE == PREFILL) {
    kvh = x % p.hkv;
    x /= p.hkv;
  } else {
    kvh = x / p.tiles;
    x -= kvh * p.tiles;
    split = kvh / p.hkv;
    kvh -= split * p.hkv;
  }
  int seq, tile, start, n, kv_len;
  if (!packed_tile<MODE>(p, x, seq, tile, start, n, kv_len)) return;
  const int q0 = tile * p.tile_tokens;
  const int tile_rows = min(p.tile_tokens, n - q0) * p.group;        // rows of this tile that exist
  const int hist = kv_len - (MODE == PREFILL ? load_index(p.q_lens, seq, p.qlens_is_int64) : 0);
  const int keys = (int)max((int64_t)0, min((int64_t)kv_len, (int64_t)p.max_pages << p.page_shift));
  // positions of the tile's first and last token; the keys that some row sees are [vis_lo, vis_hi) and those below sinks
  int vis_lo = 0, vis_hi = keys, pos_hi = 0, sink_blocks = 0, first_block, nb;
  if (MODE == PREFILL) {
    pos_hi = hist + min(q0 + p.tile_tokens, n) - 1;
    vis_lo = max(0, hist + q0 - p.window);
    vis_hi = max(0, min(keys, pos_hi + 1));
    first_block = vis_lo / BN;
    sink_blocks = min((min(p.sinks, vis_hi) + BN - 1) / BN, first_block);
    nb = max(0, (vis_hi + BN - 1) / BN - first_block);
    nb = nb > 0 ? nb + sink_blocks : 0;
  } else {
    if (split * p.prefix.chunk >= keys) return;
    first_block = split * (p.prefix.chunk / BN);
    nb = (min(p.prefix.chunk, keys - split * p.prefix.chunk) + BN - 1) / BN;
  }
  // first key of the tile's block j
  auto block_key = [&](int j) {
    return (MODE == PREFILL ? (j < sink_blocks ? j : first_block + j - sink_blocks) : first_block + j) * BN;
  };
  // does some row of the tile see one of the keys [from, to)?
  auto seen = [&](int from, int to) {
    return (from < vis_hi && to > vis_lo) || (MODE == PREFILL && from < min(p.sinks, vis_hi));
  };

  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023u) != 0) {
    // the 128-byte swizzle needs 1 KiB aligned tiles; report instead of computing garbage
    if (threadIdx.x == 0 && p.status != nullptr && atomicCAS(p.status, DLB_DEV_OK, DLB_DEV_WAIT_TIMEOUT) == DLB_DEV_OK)
      p.status[1] = 50;
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + OFF_CTRL);
  uint64_t* q_full = bars + 0;
  uint64_t* k_full = bars + 1;     // [2]
  uint64_t* v_full = bars + 3;     // [2]
  uint64_t* s_full = bars + 5;     // [2] S_j done; K stage reusable
  uint64_t* p_full = bars + 7;     // [2] P_j written
  uint64_t* pv_done = bars + 9;    // [2] P_j V_j done; V stage reusable, O updated
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 11);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  if (warp == WARP_TMA && lane == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&pv_done[i], 1);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == WARP_MMA) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t tmem_o = tmem_base + 128;

  if (warp == WARP_TMA) {
    // ------------------------------ TMA producer ------------------------------
    if (lane == 0 && nb > 0) {
      tma_prefetch_desc(&tmap_q);
      tma_prefetch_desc(&tmap_k);
      tma_prefetch_desc(&tmap_v);
      mbar_arrive_expect_tx(q_full, BOXES * p.group * p.tile_tokens * 128);
#pragma unroll
      for (int bx = 0; bx < BOXES; ++bx)
        tma_load_3d(smem + OFF_Q + bx * Q_BOX, &tmap_q, q_full, bx * 64, kvh * p.group, start + q0);
      const int box_shift = min(p.page_shift, 6);
      const int n_box = BN >> box_shift;
      // Pages of a block, at most four; -1: no key of it is seen, nothing is fetched.  The look-up of block j + 1 runs
      // behind the loads of block j, so that its latency is not between a freed stage and the next load.
      int pg[4] = {-1, -1, -1, -1};
      auto look_up = [&](int j) {
        const int key0 = block_key(j);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (u >= n_box) break;
          const int tok = key0 + (u << box_shift);
          pg[u] = -1;
          if (!seen(tok, tok + (1 << box_shift))) continue;
          const int column = tok >> p.page_shift;
          int page = load_index(p.block_table, (int64_t)seq * p.bt_stride + column, p.table_is_int64);
          if (page < 0 || page >= p.num_pages) {
            report_bad_page(p.status, seq, column, page);
            page = 0;
          }
          pg[u] = page;
        }
      };
      auto load_block = [&](int j, int off, const CUtensorMap* tmap, uint64_t* full, const int (&page)[4]) {
        uint8_t* dst = smem + off + (j & 1) * KV_BYTES;
        const int key0 = block_key(j);
        int boxes = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) boxes += u < n_box && page[u] >= 0 ? 1 : 0;
        mbar_arrive_expect_tx(&full[j & 1], (uint32_t)((boxes << box_shift) * 128 * BOXES));
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (u >= n_box || page[u] < 0) continue;
          const int slot = (key0 + (u << box_shift)) & ((1 << p.page_shift) - 1);
#pragma unroll
          for (int bx = 0; bx < BOXES; ++bx)
            tma_load_4d(dst + bx * KV_BOX + (u << box_shift) * 128, tmap, &full[j & 1], bx * 64, kvh, slot, page[u]);
        }
      };
      look_up(0);
      for (int j = 0; j < nb; ++j) {
        const int s = j & 1;
        const uint32_t ph = (j >> 1) & 1;
        int pv[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) pv[u] = pg[u];
        if (!mbar_wait(&s_full[s], ph ^ 1, abort_flag, p.status, 51, j)) break;
        load_block(j, OFF_K, &tmap_k, k_full, pg);
        if (j + 1 < nb) look_up(j + 1);
        if (!mbar_wait(&pv_done[s], ph ^ 1, abort_flag, p.status, 52, j)) break;
        load_block(j, OFF_V, &tmap_v, v_full, pv);
      }
    }
  } else if (warp == WARP_MMA) {
    // ------------------------------ MMA issuer ------------------------------
    if (lane == 0 && nb > 0) {
      bool ok = mbar_wait(q_full, 0, abort_flag, p.status, 53, 0);
      const uint64_t q_d0 = make_smem_desc(smem_u32(smem + OFF_Q), 16, 1024, 2);
      const uint64_t k_d0 = make_smem_desc(smem_u32(smem + OFF_K), 16, 1024, 2);
      // V as an MN-major operand: 64 columns contiguous, the next 64 a box further (LBO), 8 keys at 128 B, the next 8 at SBO
      const uint64_t v_d0 = make_smem_desc(smem_u32(smem + OFF_V), KV_BOX, 1024, 2);
      const uint32_t q_lo0 = (uint32_t)q_d0, k_lo0 = (uint32_t)k_d0, kq_hi = (uint32_t)(q_d0 >> 32);
      const uint32_t v_lo0 = (uint32_t)v_d0, v_hi = (uint32_t)(v_d0 >> 32);
      for (int j = 0; ok && j <= nb; ++j) {
        if (j < nb) {
          // S_j = Q K_j^T.  S buffer s also carried P_{j-2}: P_{j-2} V_{j-2} was issued before, and one thread's MMAs run in order
          const int s = j & 1;
          if (!mbar_wait(&k_full[s], (j >> 1) & 1, abort_flag, p.status, 54, j)) break;
          tc_fence_after_sync();
          const uint32_t k_lo = k_lo0 + (uint32_t)s * (KV_BYTES >> 4);
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            const uint32_t qoff = (uint32_t)(((ks >> 2) * Q_BOX + (ks & 3) * 32) >> 4);
            const uint32_t koff = (uint32_t)(((ks >> 2) * KV_BOX + (ks & 3) * 32) >> 4);
            if (ks == 0) umma_ss_lohi<0>(tmem_base + s * BN, q_lo0 + qoff, kq_hi, k_lo + koff, kq_hi, p.idesc_qk);
            else umma_ss_lohi<1>(tmem_base + s * BN, q_lo0 + qoff, kq_hi, k_lo + koff, kq_hi, p.idesc_qk);
          }
          umma_commit(&s_full[s]);
        }
        if (j > 0) {
          // O += P_{j-1} V_{j-1}
          const int jj = j - 1, s = jj & 1;
          const uint32_t ph = (jj >> 1) & 1;
          const bool r1 = mbar_try_wait(&p_full[s], ph), r2 = mbar_try_wait(&v_full[s], ph);
          if (!(r1 && r2)) {
            if (!mbar_wait(&p_full[s], ph, abort_flag, p.status, 56, jj)) break;
            if (!mbar_wait(&v_full[s], ph, abort_flag, p.status, 57, jj)) break;
          }
          tc_fence_after_sync();
          const uint32_t v_lo = v_lo0 + (uint32_t)s * (KV_BYTES >> 4);
          if (jj == 0) umma_ts_lohi<0>(tmem_o, tmem_base + s * BN, v_lo, v_hi, p.idesc_pv);
          else umma_ts_lohi<1>(tmem_o, tmem_base + s * BN, v_lo, v_hi, p.idesc_pv);
#pragma unroll
          for (int ks = 1; ks < BN / 16; ++ks)
            umma_ts_lohi<1>(tmem_o, tmem_base + s * BN + ks * 8, v_lo + ks * (16 * 128 >> 4), v_hi, p.idesc_pv);
          umma_commit(&pv_done[s]);
        }
      }
    }
  } else {
    // ------------------------------ softmax / correction / epilogue ------------------------------
    const int quad = warp;
    const int row = quad * 32 + lane;              // row of the tile == TMEM lane
    const bool live = row < tile_rows;
    const int tok = (int)((uint32_t)row * p.group_inv >> 16);
    const int q_pos = hist + q0 + tok;             // position of this row's token
    const uint32_t lane_field = (uint32_t)(quad * 32) << 16;
    float m_ref = -CUDART_INF_F;                   // reference maximum (scaled, base-2 domain)
    float l_sum = 0.f;
    bool ok = true;
    for (int j = 0; j < nb; ++j) {
      const int s = j & 1;
      const uint32_t ph = (j >> 1) & 1;
      ok = mbar_wait(&s_full[s], ph, abort_flag, p.status, 58, j);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after_sync();
      uint32_t sr[2][32];
      tmem_ld_32x32b_x32(tmem_base + lane_field + s * BN, sr[0]);
      tmem_ld_32x32b_x32(tmem_base + lane_field + s * BN + 32, sr[1]);
      tmem_wait_ld();

      float eff_scale = p.scale_log2;
      if (CAP) {
        const float inv = p.sm_scale / p.softcap, cap = p.softcap * 1.4426950408889634f;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < 32; ++c) sr[h][c] = __float_as_uint(cap * tanhf(__uint_as_float(sr[h][c]) * inv));
        eff_scale = 1.f;
      }
      const int key0 = block_key(j);
      // blocks that some row sees only in part: one bit per key of this row
      const bool whole = MODE == PREFILL ? key0 + BN - 1 <= hist + q0 && key0 + BN <= keys && key0 >= pos_hi - p.window
                                         : key0 + BN <= keys;
      if (!whole) {
        const int hi = MODE == PREFILL ? min(q_pos, keys - 1) - key0 : keys - 1 - key0;      // last visible key
        uint64_t bits = hi < 0 ? 0ull : hi >= BN - 1 ? ~0ull : (2ull << hi) - 1;
        if (MODE == PREFILL) {
          const int lo = q_pos - p.window - key0, sk = p.sinks - key0;
          const uint64_t win = lo <= 0 ? ~0ull : lo >= BN ? 0ull : ~0ull << lo;
          const uint64_t snk = sk <= 0 ? 0ull : sk >= BN ? ~0ull : (1ull << sk) - 1;
          bits &= win | snk;
        }
        const uint32_t word[2] = {(uint32_t)bits, (uint32_t)(bits >> 32)};
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (!(word[h] >> c & 1u)) sr[h][c] = 0xff800000u;   // -inf
      }
      float mx4[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};   // 4 independent chains
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int c = 0; c < 32; c += 8) {
#pragma unroll
          for (int u = 0; u < 4; ++u)
            mx4[u] = max3(mx4[u], __uint_as_float(sr[h][c + 2 * u]), __uint_as_float(sr[h][c + 2 * u + 1]));
        }
      }
      float mx = fmaxf(max3(mx4[0], mx4[1], mx4[2]), mx4[3]);
      mx = live ? mx * eff_scale : -CUDART_INF_F;     // rows past the tile's last token never ask for a rescale
      float alpha = 1.f;
      bool rescale = false;
      if (m_ref == -CUDART_INF_F) {
        m_ref = mx;                                 // first visible block: nothing accumulated yet
      } else if (mx - m_ref > RESCALE_THRESHOLD) {
        alpha = fast_exp2(m_ref - mx);
        m_ref = mx;
        rescale = true;
      }
      // O may be rescaled only once P_{j-1} V_{j-1} has retired.  (P_{j-2} V_{j-2} retired before S_j was
      // signalled, so the barrier is never more than one phase behind and the parity wait is exact.)
      if (j > 0 && __any_sync(0xffffffffu, rescale)) {
        ok = mbar_wait(&pv_done[(j - 1) & 1], ((j - 1) >> 1) & 1, abort_flag, p.status, 59, j);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after_sync();
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(tmem_o + lane_field + c * 32, o);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
          tmem_st_32x32b_x32(tmem_o + lane_field + c * 32, o);
        }
        tmem_wait_st();
      }
      // p = 2^(s * scale - m), written back as 16-bit pairs over the first columns of the S buffer it came from
      const float neg_m = (m_ref == -CUDART_INF_F) ? 0.f : -m_ref;
      const uint64_t scale2 = pack_f2(eff_scale, eff_scale);
      const uint64_t negm2 = pack_f2(neg_m, neg_m);
      uint64_t sum2a = pack_f2(0.f, 0.f), sum2b = sum2a;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t pk[16];
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          const uint64_t a01 =
              fma_f2(pack_f2(__uint_as_float(sr[h][c]), __uint_as_float(sr[h][c + 1])), scale2, negm2);
          const uint64_t a23 =
              fma_f2(pack_f2(__uint_as_float(sr[h][c + 2]), __uint_as_float(sr[h][c + 3])), scale2, negm2);
          float x0, x1, x2, x3;
          unpack_f2(a01, x0, x1);
          unpack_f2(a23, x2, x3);
          const float e0 = fast_exp2(x0), e1 = fast_exp2(x1), e2 = fast_exp2(x2), e3 = fast_exp2(x3);
          sum2a = add_f2(sum2a, pack_f2(e0, e1));
          sum2b = add_f2(sum2b, pack_f2(e2, e3));
          typename Elem<T>::T2 v01 = Elem<T>::from_f2(e0, e1);
          typename Elem<T>::T2 v23 = Elem<T>::from_f2(e2, e3);
          pk[c / 2] = *reinterpret_cast<uint32_t*>(&v01);
          pk[c / 2 + 1] = *reinterpret_cast<uint32_t*>(&v23);
        }
        tmem_st_32x32b_x16(tmem_base + lane_field + s * BN + h * 16, pk);
      }
      {
        float a, b;
        unpack_f2(add_f2(sum2a, sum2b), a, b);
        l_sum = l_sum * alpha + (a + b);
      }
      if (!whole && !(key0 >= vis_lo && key0 + BN <= vis_hi)) {
        // V rows that no row of the tile sees (past the end, behind the window of every row, not fetched): their weights are
        // zero, but 0 x (what a reused page or an old tile left there) may be NaN.  Zeroed, and made visible to the
        // tensor core's reads, before this block's P V can be issued.
        ok = mbar_wait(&v_full[s], ph, abort_flag, p.status, 61, j);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        uint8_t* vt = smem + OFF_V + s * KV_BYTES;
        for (int i = threadIdx.x; i < BN * BOXES * 8; i += 128) {
          const int chunk = i & 7, bx = (i >> 3) % BOXES, r = (i >> 3) / BOXES;
          if (!seen(key0 + r, key0 + r + 1))
            *reinterpret_cast<uint4*>(vt + bx * KV_BOX + r * 128 + chunk * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
      }
      tmem_wait_st();
      tc_fence_before_sync();
      mbar_arrive(&p_full[s]);
    }
    if (ok && nb > 0) {
      ok = mbar_wait(&pv_done[(nb - 1) & 1], ((nb - 1) >> 1) & 1, abort_flag, p.status, 60, nb);
      ok = __all_sync(0xffffffffu, ok);
    }
    if (ok) {
      tc_fence_after_sync();
      if constexpr (MODE == PREFIX) {
        const int64_t rows_all = p.tokens * p.hq;
        const int64_t at = split * rows_all + (int64_t)(start + q0 + tok) * p.hq + kvh * p.group + (row - tok * p.group);
        float4* dst = reinterpret_cast<float4*>(p.prefix.o + at * D);
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(tmem_o + lane_field + c * 32, o);
          tmem_wait_ld();
          if (live) {
#pragma unroll
            for (int v = 0; v < 8; ++v)
              dst[c * 8 + v] = make_float4(__uint_as_float(o[4 * v]), __uint_as_float(o[4 * v + 1]),
                                           __uint_as_float(o[4 * v + 2]), __uint_as_float(o[4 * v + 3]));
          }
        }
        if (live) p.prefix.ml[at] = make_float2(m_ref, l_sum);
      } else {
        // Through the Q tile's shared memory (every Q K^T has retired; row r of O over row r of Q, same swizzle), 64
        // columns at a time, so that the lanes of a store cover whole 128-byte lines.  A row that saw no key is zero.
        const float inv_l = l_sum > 0.f ? 1.f / l_sum : 0.f;
        uint8_t* stage = smem + OFF_Q;
        const int sub = lane >> 3, cc = lane & 7;              // row of four, 16-byte chunk of its line
        T* obase = reinterpret_cast<T*>(p.out) + (int64_t)(start + q0) * p.o_st + (int64_t)kvh * p.group * p.o_sh + cc * 8;
#pragma unroll 1
        for (int c = 0; quad * 32 < tile_rows && c < D / 64; ++c) {
          uint32_t o[2][32];
          if (nb > 0) {
            tmem_ld_32x32b_x32(tmem_o + lane_field + c * 64, o[0]);
            tmem_ld_32x32b_x32(tmem_o + lane_field + c * 64 + 32, o[1]);
            tmem_wait_ld();
          }
#pragma unroll
          for (int v = 0; v < 8; ++v) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int e = (v & 3) * 8 + 2 * i;
              typename Elem<T>::T2 v2 = Elem<T>::from_f2(__uint_as_float(o[v >> 2][e]) * inv_l, __uint_as_float(o[v >> 2][e + 1]) * inv_l);
              w[i] = l_sum > 0.f ? *reinterpret_cast<uint32_t*>(&v2) : 0u;
            }
            *reinterpret_cast<uint4*>(stage + c * Q_BOX + row * 128 + ((v ^ (row & 7)) << 4)) =
                make_uint4(w[0], w[1], w[2], w[3]);
          }
          __syncwarp();
          if (c * 64 + cc * 8 < p.dv) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int r = quad * 32 + i * 4 + sub;
              if (r < tile_rows) {
                const int t = (int)((uint32_t)r * p.group_inv >> 16);
                *reinterpret_cast<uint4*>(obase + (int64_t)t * p.o_st + (int64_t)(r - t * p.group) * p.o_sh + c * 64) =
                    *reinterpret_cast<const uint4*>(stage + c * Q_BOX + r * 128 + ((cc ^ (r & 7)) << 4));
              }
            }
          }
        }
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == WARP_MMA) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

template <typename T, int D, int MODE, bool CAP>
static int launch_packed_x(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const PackedParams& p,
                           unsigned grid, cudaStream_t stream) {
  auto kern = packed_attention_kernel<T, D, MODE, CAP>;
  constexpr int SMEM = pa::Layout<D>::SMEM_BYTES;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
  if (e != cudaSuccess) {
    set_last_error("packed_attention: smem attribute: %s", cudaGetErrorString(e));
    return (int)e;
  }
  kern<<<grid, pa::THREADS, SMEM, stream>>>(tq, tk, tv, p);
  DLB_CUDA_LAUNCH_CHECK();
  return DLB_OK;
}
template <int MODE>
static int launch_packed(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const PackedParams& p, int D,
                         int dtype, unsigned grid, cudaStream_t s) {
  const bool cap = p.softcap > 0.f;
  if (dtype == DLB_DTYPE_BF16) {
    if (D == 128) return cap ? launch_packed_x<__nv_bfloat16, 128, MODE, true>(tq, tk, tv, p, grid, s)
                             : launch_packed_x<__nv_bfloat16, 128, MODE, false>(tq, tk, tv, p, grid, s);
    return cap ? launch_packed_x<__nv_bfloat16, 64, MODE, true>(tq, tk, tv, p, grid, s)
               : launch_packed_x<__nv_bfloat16, 64, MODE, false>(tq, tk, tv, p, grid, s);
  }
  if (D == 128) return cap ? launch_packed_x<__half, 128, MODE, true>(tq, tk, tv, p, grid, s)
                           : launch_packed_x<__half, 128, MODE, false>(tq, tk, tv, p, grid, s);
  return cap ? launch_packed_x<__half, 64, MODE, true>(tq, tk, tv, p, grid, s)
             : launch_packed_x<__half, 64, MODE, false>(tq, tk, tv, p, grid, s);
}

// What both entry points take: types, head sizes, cache layout.  Returns DLB_OK or an error; `width` is the tile width.
static int check_attention(const char* what, int64_t batch, int64_t tokens, int64_t hq, int64_t hkv, int64_t head_dim,
                           int64_t head_dim_v, int64_t page_size, int64_t num_pages, int64_t max_pages, float sm_scale,
                           int dtype, int& width) {
  DLB_CHECK_ARG(dtype == DLB_DTYPE_BF16 || dtype == DLB_DTYPE_F16, DLB_ERR_UNSUPPORTED, "%s: dtype %d (need fp16 or bf16)",
                what, dtype);
  DLB_CHECK_ARG(head_dim >= 8 && head_dim <= 128 && head_dim % 8 == 0 && head_dim_v >= 8 && head_dim_v <= 128 &&
                    head_dim_v % 8 == 0,
                DLB_ERR_UNSUPPORTED, "%s: head_dim %lld / %lld not supported (multiples of 8 up to 128)", what,
                (long long)head_dim, (long long)head_dim_v);
  DLB_CHECK_ARG(batch >= 0 && tokens >= 0 && hq >= 1 && hkv >= 1 && hq % hkv == 0, DLB_ERR_BAD_ARG, "%s: bad sizes", what);
  DLB_CHECK_ARG(hq / hkv <= pa::BM, DLB_ERR_UNSUPPORTED, "%s: %lld q-heads to a kv head (at most %d)", what,
                (long long)(hq / hkv), pa::BM);
  DLB_CHECK_ARG(page_size >= 16 && page_size <= 65536 && (page_size & (page_size - 1)) == 0, DLB_ERR_UNSUPPORTED,
                "%s: page size %lld must be a power of two from 16 on", what, (long long)page_size);
  DLB_CHECK_ARG(num_pages >= 1 && max_pages >= 1, DLB_ERR_BAD_ARG, "%s: empty cache or table", what);
  DLB_CHECK_ARG(num_pages < (1LL << 31) && max_pages * page_size < (1LL << 31) && tokens * hq < (1LL << 31) &&
                    batch <= 65535 && hkv * ((hq / hkv + 15) / 16) <= 65535,
                DLB_ERR_TOO_LARGE, "%s: sizes past 31 bits", what);
  // the maximum is taken before the scale is applied
  DLB_CHECK_ARG(sm_scale > 0.f, DLB_ERR_BAD_ARG, "%s: sm_scale must be positive", what);
  width = (head_dim <= 64 && head_dim_v <= 64) ? 64 : 128;
  return DLB_OK;
}

static int check_rows(const char* what, const void* q, const void* out, int64_t q_st, int64_t q_sh, int64_t o_st, int64_t o_sh) {
  DLB_CHECK_ARG((((uintptr_t)q | (uintptr_t)out) & 15) == 0 && q_st % 8 == 0 && q_sh % 8 == 0 && o_st % 8 == 0 && o_sh % 8 == 0,
                DLB_ERR_ALIGNMENT, "%s: rows of q and of the output must be 16-byte aligned", what);
  return DLB_OK;
}

static int log2_of(int64_t v) {
  int s = 0;
  while ((1LL << s) < v) ++s;
  return s;
}

static void set_shape(PackedParams& p, int64_t hq, int64_t hkv, int width, float sm_scale, float softcap, int dtype) {
  p.hq = (int)hq;
  p.hkv = (int)hkv;
  p.group = (int)(hq / hkv);
  p.tile_tokens = pa::BM / p.group;
  p.group_inv = (65536u + p.group - 1) / p.group;
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.sm_scale = sm_scale;
  p.softcap = softcap;
  const uint32_t fmt = dtype == DLB_DTYPE_BF16 ? 1u : 0u;
  p.idesc_qk = make_idesc_f16(pa::BM, pa::BN, fmt, 0u, 0u);
  p.idesc_pv = make_idesc_f16(pa::BM, width, fmt, 0u, 1u);
}

}  // namespace dlb

extern "C" int dlb_sink_attention(const void* q, const void* k_cache, const void* v_cache, void* out,
                                  const void* block_table, const void* q_start_loc, const void* q_seq_len,
                                  const void* kv_seq_len, int64_t batch, int64_t total_q_tokens, int64_t max_q_len,
                                  int64_t hq, int64_t hkv, int64_t head_dim, int64_t head_dim_v, int64_t page_size,
                                  int64_t num_pages, int64_t max_pages, int64_t q_stride_t, int64_t q_stride_h,
                                  int64_t o_stride_t, int64_t o_stride_h, int64_t k_stride_page, int64_t k_stride_slot,
                                  int64_t k_stride_head, int64_t v_stride_page, int64_t v_stride_slot,
                                  int64_t v_stride_head, int64_t bt_stride, int table_is_int64, int start_is_int64,
                                  int qlen_is_int64, int kvlen_is_int64, int64_t window, int64_t sinks, float sm_scale,
                                  float softcap, int dtype, int32_t* status, void* stream) {
  DLB_NVTX("dlb_sink_attention");
  using namespace dlb;
  int width = 0;
  int rc = check_attention("sink_attention", batch, total_q_tokens, hq, hkv, head_dim, head_dim_v, page_size, num_pages,
                           max_pages, sm_scale, dtype, width);
  if (rc != DLB_OK) return rc;
  DLB_CHECK_ARG(window >= 0 && sinks >= 0 && max_q_len >= 0, DLB_ERR_BAD_ARG, "sink_attention: negative window, sinks or length");
  if (batch == 0 || total_q_tokens == 0 || max_q_len == 0) return DLB_OK;
  DLB_CHECK_ARG(q && k_cache && v_cache && out && block_table && q_start_loc && q_seq_len && kv_seq_len, DLB_ERR_BAD_ARG,
                "sink_attention: null pointer");
  rc = check_rows("sink_attention", q, out, q_stride_t, q_stride_h, o_stride_t, o_stride_h);
  if (rc != DLB_OK) return rc;
  const int win = (int)(window < (1 << 30) ? window : (1 << 30)), snk = (int)(sinks < (1 << 30) ? sinks : (1 << 30));
  cudaStream_t s = (cudaStream_t)stream;
  if (max_q_len == 1) {
    ClusterDecodeParams d = {};
    d.q = q; d.out = out; d.block_table = block_table; d.kv_lens = kv_seq_len; d.q_start = q_start_loc; d.q_lens = q_seq_len;
    d.q_st = q_stride_t; d.q_sh = q_stride_h; d.o_st = o_stride_t; d.o_sh = o_stride_h; d.bt_stride = bt_stride;
    d.tokens = total_q_tokens;
    d.batch = (int)batch; d.hq = (int)hq; d.hkv = (int)hkv; d.group = (int)(hq / hkv); d.dk = (int)head_dim; d.dv = (int)head_dim_v;
    d.page_shift = log2_of(page_size); d.max_pages = (int)max_pages; d.num_pages = (int)num_pages;
    d.table_is_int64 = table_is_int64; d.lens_is_int64 = kvlen_is_int64; d.start_is_int64 = start_is_int64; d.qlens_is_int64 = qlen_is_int64;
    d.window = win; d.sinks = snk; d.sm_scale = sm_scale; d.softcap = softcap; d.status = status;
    const int64_t bound = window + sinks + 1 < max_pages * page_size ? window + sinks + 1 : max_pages * page_size;
    return launch_cluster_decode(d, k_cache, v_cache, k_stride_page, k_stride_slot, k_stride_head, v_stride_page,
                                 v_stride_slot, v_stride_head, width, bound, dtype, s);
  }
  PackedParams p = {};
  set_shape(p, hq, hkv, width, sm_scale, softcap, dtype);
  p.out = out; p.q_start = q_start_loc; p.q_lens = q_seq_len; p.kv_lens = kv_seq_len; p.block_table = block_table;
  p.o_st = o_stride_t; p.o_sh = o_stride_h; p.bt_stride = bt_stride;
  p.tokens = total_q_tokens;
  p.batch = (int)batch;
  p.page_shift = log2_of(page_size); p.max_pages = (int)max_pages; p.num_pages = (int)num_pages; p.dv = (int)head_dim_v;
  p.table_is_int64 = table_is_int64; p.start_is_int64 = start_is_int64; p.qlens_is_int64 = qlen_is_int64; p.lens_is_int64 = kvlen_is_int64;
  p.window = win; p.sinks = snk; p.status = status;
  const int64_t tiles = total_q_tokens / p.tile_tokens + batch;      // sequences end inside a tile at most once each
  DLB_CHECK_ARG(tiles * hkv < (1LL << 31), DLB_ERR_TOO_LARGE, "sink_attention: grid too large");
  p.tiles = (int)tiles;
  CUtensorMap tq, tk, tv;
  rc = make_tmap_tokens(&tq, q, head_dim, hq, total_q_tokens, q_stride_h, q_stride_t, p.tile_tokens, p.group);
  if (rc != DLB_OK) return rc;
  const int box = (int)(page_size < pa::BN ? page_size : pa::BN);
  rc = make_tmap_cache(&tk, k_cache, head_dim, hkv, page_size, num_pages, k_stride_page, k_stride_slot, k_stride_head, box);
  if (rc != DLB_OK) return rc;
  rc = make_tmap_cache(&tv, v_cache, head_dim_v, hkv, page_size, num_pages, v_stride_page, v_stride_slot, v_stride_head, box);
  if (rc != DLB_OK) return rc;
  return launch_packed<pa::PREFILL>(tq, tk, tv, p, width, dtype, (unsigned)(tiles * hkv), s);
}

extern "C" int64_t dlb_shared_prefix_workspace_floats(int64_t tokens, int64_t hq, int64_t head_dim, int64_t splits) {
  const int64_t width = head_dim <= 64 ? 64 : 128;   // the tile width the kernels run at
  return tokens * hq * splits * (width + 2);
}

extern "C" int dlb_shared_prefix_attention(
    const void* q, const void* k_cache, const void* v_cache, void* out, const void* prefix_table, const void* prefix_len,
    const void* group_start, const void* block_table, const void* kv_seq_len, float* partial, int64_t batch,
    int64_t groups, int64_t hq, int64_t hkv, int64_t head_dim, int64_t head_dim_v, int64_t page_size, int64_t num_pages,
    int64_t prefix_max_pages, int64_t max_pages, int64_t q_stride_t, int64_t q_stride_h, int64_t o_stride_t,
    int64_t o_stride_h, int64_t k_stride_page, int64_t k_stride_slot, int64_t k_stride_head, int64_t v_stride_page,
    int64_t v_stride_slot, int64_t v_stride_head, int64_t pt_stride, int64_t bt_stride, int prefix_table_is_int64,
    int prefix_len_is_int64, int group_start_is_int64, int table_is_int64, int kvlen_is_int64, int64_t chunk,
    float sm_scale, float softcap, int dtype, int32_t* status, void* stream) {
  DLB_NVTX("dlb_shared_prefix_attention");
  using namespace dlb;
  int width = 0;
  int rc = check_attention("shared_prefix_attention", batch, batch, hq, hkv, head_dim, head_dim_v, page_size, num_pages,
                           max_pages < prefix_max_pages ? max_pages : prefix_max_pages, sm_scale, dtype, width);
  if (rc != DLB_OK) return rc;
  DLB_CHECK_ARG(groups >= 1 && groups <= batch + 65535 && prefix_max_pages * page_size < (1LL << 31) &&
                    max_pages * page_size < (1LL << 31),
                DLB_ERR_TOO_LARGE, "shared_prefix_attention: number of groups or length of a table out of range");
  DLB_CHECK_ARG(chunk >= 64 && chunk % 64 == 0 && chunk < (1LL << 31), DLB_ERR_BAD_ARG,
                "shared_prefix_attention: chunk %lld must be a multiple of 64", (long long)chunk);
  if (batch == 0) return DLB_OK;
  DLB_CHECK_ARG(q && k_cache && v_cache && out && prefix_table && prefix_len && group_start && block_table && kv_seq_len &&
                    partial,
                DLB_ERR_BAD_ARG, "shared_prefix_attention: null pointer");
  DLB_CHECK_ARG(((uintptr_t)partial & 15) == 0, DLB_ERR_ALIGNMENT, "shared_prefix_attention: workspace not 16-byte aligned");
  rc = check_rows("shared_prefix_attention", q, out, q_stride_t, q_stride_h, o_stride_t, o_stride_h);
  if (rc != DLB_OK) return rc;
  const int64_t splits = (prefix_max_pages * page_size + chunk - 1) / chunk;
  cudaStream_t s = (cudaStream_t)stream;
  PackedParams p = {};
  set_shape(p, hq, hkv, width, sm_scale, softcap, dtype);
  p.block_table = prefix_table; p.bt_stride = pt_stride; p.table_is_int64 = prefix_table_is_int64;
  p.tokens = batch;
  p.batch = (int)groups;
  p.page_shift = log2_of(page_size); p.max_pages = (int)prefix_max_pages; p.num_pages = (int)num_pages; p.dv = (int)head_dim_v;
  p.status = status;
  PrefixPartials& x = p.prefix;
  x.o = partial;
  x.ml = reinterpret_cast<float2*>(partial + splits * batch * hq * width);
  x.lens = prefix_len; x.group_start = group_start;
  x.groups = (int)groups; x.lens_is_int64 = prefix_len_is_int64; x.start_is_int64 = group_start_is_int64;
  x.max_len = (int)(prefix_max_pages * page_size); x.chunk = (int)chunk;
  const int64_t tiles = batch / p.tile_tokens + (groups < batch ? groups : batch);
  DLB_CHECK_ARG(tiles * hkv * splits < (1LL << 31), DLB_ERR_TOO_LARGE, "shared_prefix_attention: grid too large");
  p.tiles = (int)tiles;
  CUtensorMap tq, tk, tv;
  rc = make_tmap_tokens(&tq, q, head_dim, hq, batch, q_stride_h, q_stride_t, p.tile_tokens, p.group);
  if (rc != DLB_OK) return rc;
  const int box = (int)(page_size < pa::BN ? page_size : pa::BN);
  rc = make_tmap_cache(&tk, k_cache, head_dim, hkv, page_size, num_pages, k_stride_page, k_stride_slot, k_stride_head, box);
  if (rc != DLB_OK) return rc;
  rc = make_tmap_cache(&tv, v_cache, head_dim_v, hkv, page_size, num_pages, v_stride_page, v_stride_slot, v_stride_head, box);
  if (rc != DLB_OK) return rc;
  rc = launch_packed<pa::PREFIX>(tq, tk, tv, p, width, dtype, (unsigned)(tiles * hkv * splits), s);
  if (rc != DLB_OK) return rc;

  ClusterDecodeParams d = {};
  d.q = q; d.out = out; d.block_table = block_table; d.kv_lens = kv_seq_len;
  d.q_st = q_stride_t; d.q_sh = q_stride_h; d.o_st = o_stride_t; d.o_sh = o_stride_h; d.bt_stride = bt_stride;
  d.tokens = batch;
  d.batch = (int)batch; d.hq = (int)hq; d.hkv = (int)hkv; d.group = (int)(hq / hkv); d.dk = (int)head_dim; d.dv = (int)head_dim_v;
  d.page_shift = p.page_shift; d.max_pages = (int)max_pages; d.num_pages = (int)num_pages;
  d.table_is_int64 = table_is_int64; d.lens_is_int64 = kvlen_is_int64;
  d.window = -1; d.sinks = 0; d.sm_scale = sm_scale; d.softcap = softcap; d.status = status;
  d.prefix = p.prefix;
  return launch_cluster_decode(d, k_cache, v_cache, k_stride_page, k_stride_slot, k_stride_head, v_stride_page,
                               v_stride_slot, v_stride_head, width, max_pages * page_size, dtype, s);
}
