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
// One CTA = one (row tile, kv head, split), two CTAs per SM (256 TMEM columns and 97 or 113 KiB each), so that one CTA's
// softmax runs beside the other's matrix instructions.  192 threads: warp 4 issues the loads (K and V tiles of 64 keys, one
// box per page, into rings of two, or of three where the rows fit half a tile: 24 sequences of 5 drafted tokens over 2048
// keys 37 -> 32 us), one lane of warp 5 the tcgen05.mma (S_j = Q K_j^T into one of two S buffers, then O += P_{j-1} V_{j-1}
// with P as the A operand from TMEM; three buffers and P_{j-2} with 64 columns), warps 0-3 the softmax, one thread per row,
// with the exponentials taken against the old maximum before the block's own is known.  The blocks of 64 keys are those of
// the sinks and then those of the window; blocks in between are skipped, and so are pages that hold no key which the tile
// sees.  Where the tiles are few, the CTAs of a cluster share a tile's blocks and join through distributed shared memory.
//
// Bound by the chain S_j -> P_j -> P V -> S_{j+2}: a softmax warp takes about 1220 clocks for a block, the way from a P
// written to the S after next 1890, with the tensor pipe 54 %, the exponential unit 56 % and the issue slots 46 % busy (one
// prompt of 8192 tokens, window 4095, 32 / 8 heads of 128: 0.40 ms).  Two prompts of 16384: 1.72 to 1.75 ms in short runs,
// 1110 TFLOP/s, 2.04 in long ones under the power limit.  Taller tiles (two of 128 rows sharing K and V, one CTA per SM),
// blocks of 128 keys, K loaded ahead of V, L2 prefetches, turns between the tiles at the exponentials and CTAs that go on to
// further tiles were measured and gave nothing or lost up to 20 %.
#include <float.h>
#include <math_constants.h>

#include "cluster_decode.cuh"

namespace dlb {

namespace pa {
constexpr int BM = 128;           // rows per CTA
constexpr int BN = 64;            // keys per block
constexpr int THREADS = 192;      // warps 0-3 softmax (TMEM quadrant = warp id), warp 4 TMA, warp 5 MMA
constexpr int WARP_TMA = 4;
constexpr int WARP_MMA = 5;
constexpr int KV_BOX = BN * 128;  // one 64-wide (128 B) column box of a K or V block
constexpr int TMEM_COLS = 256;    // S buffers of 64 columns, P over the first half of its S, then O
constexpr float RESCALE_THRESHOLD = 8.0f;   // log2 units: P stays below 2^8, well inside fp16
enum { PREFILL, PREFIX };
// ROWS of Q in shared memory, 128 or 64; the half that 64 leave free is a third pair of K and V buffers.  With 64 columns there is
// room for four pairs, and beside O for a third S, so that Q K^T runs two blocks ahead of P V (256 sequences behind 32768 tokens:
// 135 -> 126 us; prompts the same, whose softmax warps are never idle there).
template <int D, int ROWS> struct Layout {
  static constexpr int BOXES = D / 64;
  static constexpr int S_BUFS = D == 64 ? 3 : 2;
  static constexpr int STAGES = D == 64 ? 4 : ROWS == 64 ? 3 : 2;
  static constexpr int Q_BOX = ROWS * 128;                    // one 64-wide column box of the Q tile
  static constexpr int KV_BYTES = BOXES * KV_BOX;             // one K or V block
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = OFF_Q + BOXES * Q_BOX;
  static constexpr int OFF_V = OFF_K + STAGES * KV_BYTES;
  static constexpr int OFF_CTRL = OFF_V + STAGES * KV_BYTES;
  static constexpr int SMEM_BYTES = OFF_CTRL + 192;
  static_assert(OFF_V - OFF_Q >= ROWS * D * 4, "the join keeps O in 32 bits over Q and K");
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
  int cluster;                    // CTAs that share a tile's keys, a power of two
  int page_shift, max_pages, num_pages, dv;
  int k_whole, v_whole;           // a load fetches all columns of its rows (make_tmap_rows)
  int table_is_int64, start_is_int64, qlens_is_int64, lens_is_int64;
  int window, sinks;              // PREFILL
  float scale_log2, sm_scale, softcap;
  uint32_t idesc_qk, idesc_pv;
  int* status;
  PrefixPartials prefix;          // PREFIX
};

// First row, number of rows and number of keys of sequence (or group) b; rows outside q are nobody's.
template <int MODE>
__device__ __forceinline__ void packed_rows(const PackedParams& p, int b, int& start, int& n, int& kv_len) {
  if (MODE == pa::PREFIX) {
    group_rows(p.prefix, p.tokens, b, start, n);
    kv_len = clamped_index(p.prefix.lens, b, p.prefix.lens_is_int64);
  } else {
    start = clamped_index(p.q_start, b, p.start_is_int64);
    n = clamped_index(p.q_lens, b, p.qlens_is_int64);
    kv_len = clamped_index(p.kv_lens, b, p.lens_is_int64);
    n = (start < 0 || start >= p.tokens) ? 0 : (int)min((int64_t)max(n, 0), p.tokens - start);
  }
}

// Row tile x of the launch -> sequence (or group) and tile inside it, its rows and keys; false if there is none.  The tiles
// that exist are numbered through, sequence by sequence, so that a batch of any lengths needs no more CTAs than it has tiles.
// Every warp counts for itself: a lane has EACH sequences, one where 32 lanes are enough for the batch (its sizes are then at
// hand when it is found), else four, so that few loads wait for one another.
template <int MODE, int EACH>
__device__ __forceinline__ bool packed_tile(const PackedParams& p, int x, int& seq, int& tile, int& start, int& n, int& kv_len) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32 * EACH) {
    int mine[EACH], all = 0, st = 0, rows = 0, keys = 0;
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
      const int b = b0 + lane * EACH + u;
      rows = 0;
      if (b < p.batch) packed_rows<MODE>(p, b, st, rows, keys);
      mine[u] = (rows + p.tile_tokens - 1) / p.tile_tokens;
      all += mine[u];
    }
    int upto = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, before + upto > x);
    if (past != 0) {
      const int src = __ffs(past) - 1;
      int at = before + __shfl_sync(0xffffffffu, upto - all, src), of_seq = 0;     // tiles in front of the lane's first sequence
      seq = b0 + src * EACH - 1;
#pragma unroll
      for (int u = 0; u < EACH; ++u) {
        const int m = __shfl_sync(0xffffffffu, mine[u], src);
        if (at + of_seq <= x) {
          at += of_seq;
          of_seq = m;
          ++seq;
        }
      }
      tile = of_seq - 1 - (x - at);                       // the late, long ones first
      if (EACH == 1) {
        start = __shfl_sync(0xffffffffu, st, src);
        n = __shfl_sync(0xffffffffu, rows, src);
        kv_len = __shfl_sync(0xffffffffu, keys, src);
      } else {
        packed_rows<MODE>(p, seq, start, n, kv_len);
      }
      return true;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return false;
}

template <typename T, int D, int MODE, int ROWS, bool CAP>
__global__ void __launch_bounds__(pa::THREADS, 2)
packed_attention_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                        const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ PackedParams p) {
  using namespace pa;
  using L = Layout<D, ROWS>;
  constexpr int BOXES = L::BOXES, KV_BYTES = L::KV_BYTES, Q_BOX = L::Q_BOX, STAGES = L::STAGES, S_BUFS = L::S_BUFS;
  constexpr int OFF_Q = L::OFF_Q, OFF_K = L::OFF_K, OFF_V = L::OFF_V, OFF_CTRL = L::OFF_CTRL;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (warp == WARP_TMA && lane == 0) {
    tma_prefetch_desc(&tmap_q);
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  // ---- which tile: PREFILL has the kv heads of a tile side by side, PREFIX the row tiles of a (kv head, split), which
  // read the same keys; the CTAs of a cluster share one ----
  const int cluster = p.cluster, rank = (int)blockIdx.x & (cluster - 1);
  int x = (int)blockIdx.x / cluster, kvh, split = 0;
  if (MODE == PREFILL) {
    kvh = x % p.hkv;
    x /= p.hkv;
  } else {
    kvh = x / p.tiles;
    x -= kvh * p.tiles;
    split = kvh / p.hkv;
    kvh -= split * p.hkv;
  }
  if (MODE == PREFIX) let_next_start();
  int seq, tile, start, n, kv_len;
  if (!(p.batch <= 32 ? packed_tile<MODE, 1>(p, x, seq, tile, start, n, kv_len) : packed_tile<MODE, 4>(p, x, seq, tile, start, n, kv_len)))
    return;
  const int q0 = tile * p.tile_tokens;
  const int tile_rows = min(p.tile_tokens, n - q0) * p.group;        // rows of this tile that exist
  const int hist = kv_len - (MODE == PREFILL ? clamped_index(p.q_lens, seq, p.qlens_is_int64) : 0);
  const int keys = (int)max((int64_t)0, min((int64_t)kv_len, (int64_t)p.max_pages << p.page_shift));
  // positions of the tile's first and last token; the keys that some row sees are [vis_lo, vis_hi) and those below sinks
  int vis_lo = 0, vis_hi = keys, pos_hi = 0, sink_blocks = 0, first_block, nb;
  if (MODE == PREFILL) {
    pos_hi = hist + min(q0 + p.tile_tokens, n) - 1;
    vis_lo = max(0, max(0, hist + q0) - p.window);           // (a window may be as long as an int)
    vis_hi = max(0, min(keys, pos_hi + 1));
    first_block = vis_lo / BN;
    sink_blocks = min((min(p.sinks, vis_hi) + BN - 1) / BN, first_block);
    nb = sink_blocks + max(0, (vis_hi + BN - 1) / BN - first_block);
  } else {
    if (split * p.prefix.chunk >= keys) return;
    first_block = split * (p.prefix.chunk / BN);
    nb = (min(p.prefix.chunk, keys - split * p.prefix.chunk) + BN - 1) / BN;
  }
  // this CTA's blocks
  const int j_lo = nb * rank / cluster;
  nb = nb * (rank + 1) / cluster - j_lo;
  // first key of the tile's block j
  auto block_key = [&](int j) {
    j += j_lo;
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
  // block j uses the K and V buffers j % STAGES and waits for parity (j / STAGES) & 1 of their barriers; S and P have S_BUFS buffers
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + OFF_CTRL);
  uint64_t* q_full = bars + 0;
  uint64_t* k_full = bars + 1;               // [STAGES]
  uint64_t* v_full = k_full + STAGES;        // [STAGES]
  uint64_t* qk_done = v_full + STAGES;       // [STAGES] S there; K buffer reusable
  uint64_t* pv_done = qk_done + STAGES;      // [STAGES] O updated; V buffer reusable
  uint64_t* p_full = pv_done + STAGES;       // [S_BUFS] P written
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(p_full + S_BUFS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* begun = abort_flag + 1;      // [4] blocks whose K and V loads, Q K^T and P V have begun

  if (warp == WARP_TMA && lane == 0) {
    mbar_init(q_full, 1);
    for (int h = 0; h < STAGES; ++h) {
      mbar_init(&k_full[h], 1);
      mbar_init(&v_full[h], 1);
      mbar_init(&qk_done[h], 1);
      mbar_init(&pv_done[h], 1);
    }
    for (int h = 0; h < S_BUFS; ++h) mbar_init(&p_full[h], 128);
    *abort_flag = 0;
    begun[0] = begun[1] = begun[2] = begun[3] = 0;
    fence_mbar_init();
  }
  if (warp == WARP_MMA) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  // The loading warp, which set up the barriers, needs nothing of the others and does not wait for them (and the tensor memory)
  if (warp == WARP_TMA) {
    __syncwarp();
    asm volatile("bar.arrive 1, %0;" ::"n"(THREADS) : "memory");
  } else {
    tc_fence_before_sync();
    asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
    tc_fence_after_sync();
  }
  const uint32_t tmem_base = warp == WARP_TMA ? 0u : *tmem_slot;
  const uint32_t tmem_o = tmem_base + S_BUFS * BN;

  float m_ref = 0.f, l_sum = 0.f;                  // softmax warps: reference maximum (scaled, base-2 domain) and sum
  const int row = threadIdx.x;                     // row of the tile == TMEM lane
  const uint32_t lane_field = (uint32_t)(warp * 32) << 16;

  if (warp == WARP_TMA) {
    // ------------------------------ TMA producer ------------------------------
    // Lane l fetches box l of a block: 64 / min(page, 64) boxes, one page each.  The table entries of 32 boxes are asked for at
    // once, one per lane, and looked at when they come into use.  The loop is short on purpose: this warp shares its
    // scheduler with two busy softmax warps, so an instruction takes it about ten clocks, and a late load holds up everything.
    if (nb > 0) {
      if (lane == 0) {
        mbar_arrive_expect_tx(q_full, BOXES * p.group * p.tile_tokens * 128);
#pragma unroll
        for (int bx = 0; bx < BOXES; ++bx)
          tma_load_3d(smem + OFF_Q + bx * Q_BOX, &tmap_q, q_full, bx * 64, kvh * p.group, start + q0);
      }
      const int box_shift = min(p.page_shift, 6), boxes_shift = 6 - box_shift, n_box = 1 << boxes_shift;
      const int batch = 32 >> boxes_shift;                     // blocks to a batch of entries
      const uint32_t box_bytes = (uint32_t)((128 * BOXES) << box_shift);
      // first key of this lane's box of the batch from block j on; does some row see a key of it?
      auto lane_key = [&](int j) { return block_key(j + (lane >> boxes_shift)) + ((lane & (n_box - 1)) << box_shift); };
      auto wanted = [&](int j) {
        return j + (lane >> boxes_shift) < nb && seen(lane_key(j), lane_key(j) + (1 << box_shift));
      };
      auto entry = [&](int j) {
        return wanted(j) ? clamped_index(p.block_table, (int64_t)seq * p.bt_stride + (lane_key(j) >> p.page_shift), p.table_is_int64)
                         : 0;
      };
      int pages = 0, pages_next = entry(0), k_begun = 0, v_begun = 0;
      for (int j = 0; j < nb; ++j) {
        const int in_batch = j & (batch - 1);
        if (in_batch == 0) {
          pages = pages_next;
          pages_next = entry(j + batch);
          if (pages < 0 || pages >= p.num_pages) {
            report_bad_page(p.status, seq, lane_key(j) >> p.page_shift, pages);
            pages = 0;
          }
        }
        const int s = j % STAGES;
        const uint32_t ph = (j / STAGES) & 1;
        const int key = block_key(j) + (lane << box_shift);
        const bool fetch = lane < n_box && seen(key, key + (1 << box_shift));
        const int page = __shfl_sync(0xffffffffu, pages, (in_batch << boxes_shift) + (lane & (n_box - 1)));
        const int slot = key & ((1 << p.page_shift) - 1);
        uint8_t* dst = smem + s * KV_BYTES + ((lane << box_shift) & (BN - 1)) * 128;
        const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, fetch)) * box_bytes;
        auto load = [&](uint8_t* to, const CUtensorMap* map, uint64_t* full, bool whole_rows) {
          if (whole_rows) {
            tma_load_5d(to, map, full, 0, kvh, slot, 0, page);
          } else {
#pragma unroll
            for (int bx = 0; bx < BOXES; ++bx) tma_load_4d(to + bx * KV_BOX, map, full, bx * 64, kvh, slot, page);
          }
        };
        int ok = 1;
        if (lane == 0) {
          ok = mbar_wait(&qk_done[s], ph ^ 1, abort_flag, p.status, 51, j) ? 1 : 0;
          if (ok) mbar_arrive_expect_tx(&k_full[s], bytes);
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) break;
        k_begun = j + 1;
        if (fetch) load(dst + OFF_K, &tmap_k, &k_full[s], p.k_whole);
        if (lane == 0) {
          ok = mbar_wait(&pv_done[s], ph ^ 1, abort_flag, p.status, 52, j) ? 1 : 0;
          if (ok) mbar_arrive_expect_tx(&v_full[s], bytes);
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) break;
        v_begun = j + 1;
        if (fetch) load(dst + OFF_V, &tmap_v, &v_full[s], p.v_whole);
      }
      if (lane == 0) {
        begun[0] = k_begun;
        begun[1] = v_begun;
      }
    }
  } else if (warp == WARP_MMA) {
    // ------------------------------ MMA issuer ------------------------------
    // One thread's MMAs run in the order of their issue, so an S overwrites the P before it in its buffer only once P V has read that.
    if (lane == 0 && nb > 0) {
      bool ok = mbar_wait(q_full, 0, abort_flag, p.status, 53, 0);
      const uint64_t q_d0 = make_smem_desc(smem_u32(smem + OFF_Q), 16, 1024, 2);
      const uint64_t k_d0 = make_smem_desc(smem_u32(smem + OFF_K), 16, 1024, 2);
      // V as an MN-major operand: 64 columns contiguous, the next 64 a box further (LBO), 8 keys at 128 B, the next 8 at SBO
      const uint64_t v_d0 = make_smem_desc(smem_u32(smem + OFF_V), KV_BOX, 1024, 2);
      const uint32_t q_lo0 = (uint32_t)q_d0, k_lo0 = (uint32_t)k_d0, kq_hi = (uint32_t)(q_d0 >> 32);
      const uint32_t v_lo0 = (uint32_t)v_d0, v_hi = (uint32_t)(v_d0 >> 32);
      constexpr int AHEAD = S_BUFS - 1;                        // P V comes that many blocks after Q K^T
      int qk_begun = 0, pv_begun = 0;
      for (int j = 0; ok && j < nb + AHEAD; ++j) {
        if (j < nb) {
          // S_j = Q K_j^T
          const int s = j % STAGES;
          if (!mbar_wait(&k_full[s], (j / STAGES) & 1, abort_flag, p.status, 54, j)) break;
          tc_fence_after_sync();
          const uint32_t k_lo = k_lo0 + (uint32_t)s * (KV_BYTES >> 4);
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            const uint32_t qoff = (uint32_t)(((ks >> 2) * Q_BOX + (ks & 3) * 32) >> 4);
            const uint32_t koff = (uint32_t)(((ks >> 2) * KV_BOX + (ks & 3) * 32) >> 4);
            if (ks == 0) umma_ss_lohi<0>(tmem_base + (j % S_BUFS) * BN, q_lo0 + qoff, kq_hi, k_lo + koff, kq_hi, p.idesc_qk);
            else umma_ss_lohi<1>(tmem_base + (j % S_BUFS) * BN, q_lo0 + qoff, kq_hi, k_lo + koff, kq_hi, p.idesc_qk);
          }
          umma_commit(&qk_done[s]);
          qk_begun = j + 1;
        }
        if (j >= AHEAD) {
          // O += P V of block jj
          const int jj = j - AHEAD, s = jj % STAGES, u = jj % S_BUFS;
          const uint32_t p_ph = (jj / S_BUFS) & 1, v_ph = (jj / STAGES) & 1, pt = tmem_base + u * BN;
          const bool r1 = mbar_try_wait(&p_full[u], p_ph), r2 = mbar_try_wait(&v_full[s], v_ph);
          if (!(r1 && r2)) {
            if (!mbar_wait(&p_full[u], p_ph, abort_flag, p.status, 56, jj)) break;
            if (!mbar_wait(&v_full[s], v_ph, abort_flag, p.status, 57, jj)) break;
          }
          tc_fence_after_sync();
          const uint32_t v_lo = v_lo0 + (uint32_t)s * (KV_BYTES >> 4);
          if (jj == 0) umma_ts_lohi<0>(tmem_o, pt, v_lo, v_hi, p.idesc_pv);
          else umma_ts_lohi<1>(tmem_o, pt, v_lo, v_hi, p.idesc_pv);
#pragma unroll
          for (int ks = 1; ks < BN / 16; ++ks) umma_ts_lohi<1>(tmem_o, pt + ks * 8, v_lo + ks * (16 * 128 >> 4), v_hi, p.idesc_pv);
          umma_commit(&pv_done[s]);
          pv_begun = jj + 1;
        }
      }
      begun[2] = qk_begun;
      begun[3] = pv_begun;
    }
  } else {
    // ------------------------------ softmax / correction ------------------------------
    const bool live = row < tile_rows;
    const int q_pos = hist + q0 + (int)((uint32_t)row * p.group_inv >> 16);      // position of this row's token
    auto first_key = [&](int pos) { return max(0, max(0, pos) - p.window); };    // of its window
    const int q_from = first_key(q_pos);
    const float cap_in = CAP ? 2.f * 1.4426950408889634f * p.sm_scale / p.softcap : 0.f, cap_out = p.softcap * 1.4426950408889634f,
                cap_x = CAP ? p.sm_scale / p.softcap : 0.f;
    const float eff_scale = CAP ? 1.f : p.scale_log2;
    bool ok = true;
    // A warp whose rows are all past the tile's last one keeps in step and computes nothing: its P and O stay what they are, and
    // no other row reads them.
    const bool busy = warp * 32 < tile_rows;
    // what every row of the warp sees, but for the sinks; never past what the tile sees, so that a warp without rows also zeroes
    // its V rows there
    const int whole_to = min(vis_hi, hist + q0 + (int)((uint32_t)(warp * 32) * p.group_inv >> 16) + 1);
    const int whole_from = first_key(hist + q0 + (int)((uint32_t)(max(min(warp * 32 + 32, tile_rows), 1) - 1) * p.group_inv >> 16));
    for (int j = 0; j < nb; ++j) {
      const int s = j % STAGES;
      ok = mbar_wait(&qk_done[s], (j / STAGES) & 1, abort_flag, p.status, 58, j);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after_sync();
      const uint32_t s_cols = tmem_base + lane_field + (j % S_BUFS) * BN;
      const int key0 = block_key(j);
      // does every row of the warp see the whole block?
      const bool whole = MODE == PREFILL ? key0 + BN <= whole_to && (key0 >= whole_from || key0 + BN <= p.sinks) : key0 + BN <= keys;
      if (busy) {
        uint32_t sr[2][32];
        tmem_ld_32x32b_x32(s_cols, sr[0]);
        tmem_ld_32x32b_x32(s_cols + 32, sr[1]);
        tmem_wait_ld();
        // largest score of the row, three at a time in four chains
        auto largest = [&] {
          float m4[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int c = 0; c < 32; c += 8) {
#pragma unroll
              for (int u = 0; u < 4; ++u)
                m4[u] = max3(m4[u], __uint_as_float(sr[h][c + 2 * u]), __uint_as_float(sr[h][c + 2 * u + 1]));
            }
          }
          return fmaxf(max3(m4[0], m4[1], m4[2]), m4[3]);
        };
        // one bit per key of this row that it sees
        uint32_t word[2] = {~0u, ~0u};
        if (!whole) {
          const int hi = MODE == PREFILL ? min(q_pos, keys - 1) - key0 : keys - 1 - key0;      // last visible key
          uint64_t bits = hi < 0 ? 0ull : hi >= BN - 1 ? ~0ull : (2ull << hi) - 1;
          if (MODE == PREFILL) {
            const int lo = q_from - key0, sk = p.sinks - key0;
            const uint64_t win = lo <= 0 ? ~0ull : lo >= BN ? 0ull : ~0ull << lo;
            const uint64_t snk = sk <= 0 ? 0ull : sk >= BN ? ~0ull : (1ull << sk) - 1;
            bits &= win | snk;
          }
          word[0] = (uint32_t)bits;
          word[1] = (uint32_t)(bits >> 32);
        }
        auto hide = [&](uint32_t as) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (!(word[h] >> c & 1u)) sr[h][c] = as;
        };
        float mx = 0.f;
        if (CAP) {
          // Scores below the cap, which they nearly always are, go through a polynomial, a short one below a quarter of it: the
          // exponential and the reciprocal of the other way take the special-function unit twice as long as the softmax itself
          // (chunks of 7 prompts 157 -> 139 -> 131 us).  Keys out of sight are anything here, and may lead the longer way.
          float m4[4] = {CUDART_INF_F, CUDART_INF_F, CUDART_INF_F, CUDART_INF_F};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int c = 0; c < 32; c += 8) {
#pragma unroll
              for (int u = 0; u < 4; ++u)
                m4[u] = min3(m4[u], __uint_as_float(sr[h][c + 2 * u]), __uint_as_float(sr[h][c + 2 * u + 1]));
            }
          }
          mx = largest();
          const float size = fmaxf(mx, -fminf(min3(m4[0], m4[1], m4[2]), m4[3]));
          auto each_pair = [&](auto&& f) {
            float unused;
            unpack_f2(f(pack_f2(mx, mx)), mx, unused);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int c = 0; c < 32; c += 2) {
                float a, b;
                unpack_f2(f(pack_f2(__uint_as_float(sr[h][c]), __uint_as_float(sr[h][c + 1]))), a, b);
                sr[h][c] = __float_as_uint(a);
                sr[h][c + 1] = __float_as_uint(b);
              }
          };
          const SoftCapShort cap_short(cap_x, p.scale_log2);
          if (!__any_sync(0xffffffffu, live && !(size * cap_x <= 0.25f))) {
            each_pair(cap_short);
          } else if (!__any_sync(0xffffffffu, live && !(size * cap_x <= 1.f))) {
            const uint64_t x2 = pack_f2(cap_x, cap_x), out2 = pack_f2(p.scale_log2, p.scale_log2);
            each_pair([&](uint64_t v) { return soft_cap_below(v, x2, out2); });
          } else {
            each_pair([&](uint64_t v) {
              float a, b;
              unpack_f2(v, a, b);
              soft_cap_any(a, b, cap_short, cap_x, cap_in, cap_out);
              return pack_f2(a, b);
            });
          }
        }
        if (!whole) hide(0xff800000u);                // -inf
        // p = 2^(s * scale - m) as 16-bit pairs, and their sum
        uint32_t pk[2][16];
        auto weigh = [&](float m) {
          const uint64_t scale2 = pack_f2(eff_scale, eff_scale);
          const float neg = m == -CUDART_INF_F ? 0.f : -m;
          const uint64_t negm2 = pack_f2(neg, neg);
          uint64_t sum2a = pack_f2(0.f, 0.f), sum2b = sum2a;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
              const uint64_t a01 = fma_f2(pack_f2(__uint_as_float(sr[h][c]), __uint_as_float(sr[h][c + 1])), scale2, negm2);
              const uint64_t a23 = fma_f2(pack_f2(__uint_as_float(sr[h][c + 2]), __uint_as_float(sr[h][c + 3])), scale2, negm2);
              float x0, x1, x2, x3;
              unpack_f2(a01, x0, x1);
              unpack_f2(a23, x2, x3);
              const float e0 = fast_exp2(x0), e1 = fast_exp2(x1), e2 = fast_exp2(x2), e3 = fast_exp2(x3);
              sum2a = add_f2(sum2a, pack_f2(e0, e1));
              sum2b = add_f2(sum2b, pack_f2(e2, e3));
              typename Elem<T>::T2 v01 = Elem<T>::from_f2(e0, e1);
              typename Elem<T>::T2 v23 = Elem<T>::from_f2(e2, e3);
              pk[h][c / 2] = *reinterpret_cast<uint32_t*>(&v01);
              pk[h][c / 2 + 1] = *reinterpret_cast<uint32_t*>(&v23);
            }
          }
          float a, b;
          unpack_f2(add_f2(sum2a, sum2b), a, b);
          return a + b;
        };
        // With the reference as it is, which nearly always stays: so the exponentials do not wait for this block's maximum
        float sum = weigh(m_ref);
        if (!CAP || !whole) mx = largest() * eff_scale;
        if (!live) mx = -CUDART_INF_F;                  // rows past the tile's last token never ask for more
        bool raise = mx - m_ref > RESCALE_THRESHOLD;
        if (j == 0) {
          // It starts at 0 and stays there if the row's first maximum lies in [0, 8], so that the largest P is 1 or more (one
          // exponential pass less for a tile: chunks with a window of 64 94 -> 91 us); -inf until a row has seen a key.
          raise |= mx < 0.f && mx > -CUDART_INF_F;
          if (mx == -CUDART_INF_F) m_ref = mx;
        }
        if (__any_sync(0xffffffffu, raise)) {
          const bool scale_o = j > 0 && __any_sync(0xffffffffu, raise && m_ref > -CUDART_INF_F);      // else O is nothing yet
          const float alpha = raise ? fast_exp2(m_ref - mx) : 1.f;
          if (raise) m_ref = mx;
          if (scale_o) {
            // O may be rescaled only once P_{j-1} V_{j-1} has retired (its barrier completes again only with a later block's P V,
            // which waits for this one's P: the parity is exact).
            ok = mbar_wait(&pv_done[(j - 1) % STAGES], ((j - 1) / STAGES) & 1, abort_flag, p.status, 59, j);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after_sync();
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld_32x32b_x32(tmem_o + lane_field + c * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int u = 0; u < 32; ++u) o[u] = __float_as_uint(__uint_as_float(o[u]) * alpha);
              tmem_st_32x32b_x32(tmem_o + lane_field + c * 32, o);
            }
            tmem_wait_st();
          }
          if (j > 0) l_sum *= alpha;
          sum = weigh(m_ref);
        }
        l_sum += sum;
        // over the first columns of the block's S
        tmem_st_32x32b_x16(s_cols, pk[0]);
        tmem_st_32x32b_x16(s_cols + 16, pk[1]);
      }
      if (!whole && !(key0 >= vis_lo && key0 + BN <= vis_hi) && !(MODE == PREFILL && key0 + BN <= min(p.sinks, vis_hi))) {
        // V rows that no row of the tile sees (past the end, behind the window of every row, not fetched): their weights
        // are zero, but 0 x (what a reused page or an old tile left there) may be NaN.  Zeroed, and made visible to the
        // tensor core's reads, before this block's P V can be issued.  Two threads to a row.
        const int r = threadIdx.x >> 1;
        if (!seen(key0 + r, key0 + r + 1)) {
          ok = mbar_wait(&v_full[s], (j / STAGES) & 1, abort_flag, p.status, 61, j);
          uint8_t* vt = smem + OFF_V + s * KV_BYTES + r * 128;
#pragma unroll
          for (int u = 0; u < BOXES * 4; ++u)
            *reinterpret_cast<uint4*>(vt + (u >> 2) * KV_BOX + (((threadIdx.x & 1) * 4 + (u & 3) + r) & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
          fence_proxy_async_smem();
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
      tmem_wait_st();
      tc_fence_before_sync();
      mbar_arrive(&p_full[j % S_BUFS]);
    }
    if (ok && nb > 0) {
      ok = mbar_wait(&pv_done[(nb - 1) % STAGES], ((nb - 1) / STAGES) & 1, abort_flag, p.status, 60, nb);
      ok = __all_sync(0xffffffffu, ok);
    }
    tc_fence_after_sync();
    if (MODE == PREFIX || cluster > 1) {
      // O in 32 bits over Q and K (every MMA has retired), 16-byte chunk q of row r at q ^ (r & 7); maximum and sum over V
      float* ml = reinterpret_cast<float*>(smem + OFF_V);
      ml[row] = ok ? m_ref : -CUDART_INF_F;
      ml[BM + row] = ok ? l_sum : 0.f;
#pragma unroll 1
      for (int c = 0; ok && busy && nb > 0 && c < D / 32; ++c) {
        uint32_t o[32];
        tmem_ld_32x32b_x32(tmem_o + lane_field + c * 32, o);
        tmem_wait_ld();
#pragma unroll
        for (int v = 0; v < 8; ++v)
          *reinterpret_cast<uint4*>(smem + OFF_Q + row * (D * 4) + (((c * 8 + v) ^ (row & 7)) << 4)) =
              make_uint4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
      }
    } else if (ok) {
      // Through the Q tile's shared memory (every Q K^T has retired; row r of O over row r of Q, same swizzle), 64
      // columns at a time, so that the lanes of a store cover whole 128-byte lines.  A row that saw no key is zero.
      const float inv_l = 1.f / l_sum;
      uint8_t* stage = smem + OFF_Q;
      const int sub = lane >> 3, cc = lane & 7;              // row of four, 16-byte chunk of its line
      T* obase = reinterpret_cast<T*>(p.out) + (int64_t)(start + q0) * p.o_st + (int64_t)kvh * p.group * p.o_sh + cc * 8;
#pragma unroll 1
      for (int c = 0; busy && c < D / 64; ++c) {
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
          for (int u = 0; u < 4; ++u) {
            const int e = (v & 3) * 8 + 2 * u;
            typename Elem<T>::T2 v2 = Elem<T>::from_f2(__uint_as_float(o[v >> 2][e]) * inv_l, __uint_as_float(o[v >> 2][e + 1]) * inv_l);
            w[u] = l_sum == 0.f ? 0u : *reinterpret_cast<uint32_t*>(&v2);
          }
          *reinterpret_cast<uint4*>(stage + c * Q_BOX + row * 128 + ((v ^ (row & 7)) << 4)) =
              make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncwarp();
        if (c * 64 + cc * 8 < p.dv) {
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const int r = warp * 32 + u * 4 + sub;
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

  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0) {
      if (nb > 0) settle_ring(q_full, 1, 1);
      settle_ring(k_full, STAGES, begun[0]);
      settle_ring(v_full, STAGES, begun[1]);
      settle_ring(qk_done, STAGES, begun[2]);
      settle_ring(pv_done, STAGES, begun[3]);
    }
    __syncthreads();
  }
  if (warp == WARP_MMA) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
  if (MODE == PREFILL && cluster == 1) return;

  // ------------------------------ join the cluster ------------------------------
  // Each CTA takes its share of the rows from all of them, four columns at a time.
  if (cluster > 1) cluster_barrier();
  constexpr int QUADS = D / 4;
  const uint32_t at_o = smem_u32(smem + OFF_Q), at_m = smem_u32(smem + OFF_V), at_l = at_m + BM * 4;
  const int r_lo = tile_rows * rank / cluster, r_hi = tile_rows * (rank + 1) / cluster;
  for (int idx = threadIdx.x; idx < (r_hi - r_lo) * QUADS; idx += THREADS) {
    const int r = r_lo + idx / QUADS, q = idx % QUADS;
    Joined j;
    for (int c0 = 0; c0 < cluster; c0 += 4) {      // four pieces under way together
      float m[4], l[4];
      float4 o[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int c = min(c0 + u, cluster - 1);
        m[u] = peer_load(peer_address(at_m + r * 4, c));
        l[u] = peer_load(peer_address(at_l + r * 4, c));
        o[u] = peer_load4(peer_address(at_o + r * (D * 4) + ((q ^ (r & 7)) << 4), c));
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (c0 + u < cluster) j.add(m[u], l[u], o[u]);
    }
    const int t = (int)((uint32_t)r * p.group_inv >> 16);
    const int64_t token = start + q0 + t, head = kvh * p.group + (r - t * p.group);
    if constexpr (MODE == PREFIX) {
      const int64_t at = (split * p.tokens + token) * p.hq + head;
      *reinterpret_cast<float4*>(p.prefix.o + at * D + q * 4) = j.o;
      if (q == 0) p.prefix.ml[at] = make_float2(j.m, j.l);
    } else {
      store_joined<T>(reinterpret_cast<T*>(p.out) + token * p.o_st + head * p.o_sh, q * 4, p.dv, j);
    }
  }
  if (cluster > 1) cluster_barrier();    // a CTA's shared memory stays until its peers have read it
}

template <typename T, int D, int MODE, int ROWS, bool CAP>
static int launch_packed_x(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const PackedParams& p,
                           unsigned grid, cudaStream_t stream) {
  return launch_in_clusters<packed_attention_kernel<T, D, MODE, ROWS, CAP>>("packed_attention", dim3(grid * p.cluster), pa::THREADS,
                                                                            pa::Layout<D, ROWS>::SMEM_BYTES, p.cluster, false,
                                                                            stream, tq, tk, tv, p);
}
template <typename T, int D, int MODE>
static int launch_packed_x(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const PackedParams& p,
                           unsigned grid, cudaStream_t s) {
  const bool cap = p.softcap > 0.f;
  if (p.tile_tokens * p.group <= 64)
    return cap ? launch_packed_x<T, D, MODE, 64, true>(tq, tk, tv, p, grid, s)
               : launch_packed_x<T, D, MODE, 64, false>(tq, tk, tv, p, grid, s);
  return cap ? launch_packed_x<T, D, MODE, 128, true>(tq, tk, tv, p, grid, s)
             : launch_packed_x<T, D, MODE, 128, false>(tq, tk, tv, p, grid, s);
}
template <int MODE>
static int launch_packed(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const PackedParams& p, int D,
                         int dtype, unsigned grid, cudaStream_t s) {
  if (dtype == DLB_DTYPE_BF16)
    return D == 128 ? launch_packed_x<__nv_bfloat16, 128, MODE>(tq, tk, tv, p, grid, s)
                    : launch_packed_x<__nv_bfloat16, 64, MODE>(tq, tk, tv, p, grid, s);
  return D == 128 ? launch_packed_x<__half, 128, MODE>(tq, tk, tv, p, grid, s)
                  : launch_packed_x<__half, 64, MODE>(tq, tk, tv, p, grid, s);
}

// Keys are counted in 32 bits, by the loading warps up to 64 blocks of 64 past the last one.
static bool too_long(int64_t max_pages, int64_t page_size) {
  return max_pages >= (1LL << 31) || max_pages * page_size > INT_MAX - 8192;
}

// What both entry points take: types, head sizes, cache layout.  Returns DLB_OK or an error; `width` is the tile width.
static int check_attention(const char* what, int64_t batch, int64_t tokens, int64_t hq, int64_t hkv, int64_t head_dim,
                           int64_t head_dim_v, int64_t page_size, int64_t num_pages, int64_t max_pages, float sm_scale,
                           float& softcap, int dtype, int& width) {
  DLB_CHECK_ARG(dtype == DLB_DTYPE_BF16 || dtype == DLB_DTYPE_F16, DLB_ERR_UNSUPPORTED, "%s: dtype %d (need fp16 or bf16)",
                what, dtype);
  DLB_CHECK_ARG(head_dim >= 8 && head_dim <= 128 && head_dim % 8 == 0 && head_dim_v >= 8 && head_dim_v <= 128 &&
                    head_dim_v % 8 == 0,
                DLB_ERR_UNSUPPORTED, "%s: head_dim %lld / %lld not supported (multiples of 8 up to 128)", what,
                (long long)head_dim, (long long)head_dim_v);
  DLB_CHECK_ARG(batch >= 0 && tokens >= 0 && hq >= 1 && hkv >= 1 && hq % hkv == 0, DLB_ERR_BAD_ARG, "%s: bad sizes", what);
  DLB_CHECK_ARG(hq / hkv <= pa::BM, DLB_ERR_UNSUPPORTED, "%s: %lld q-heads to a kv head (at most %d)", what,
                (long long)(hq / hkv), pa::BM);
  DLB_CHECK_ARG(page_size >= 16 && page_size <= (1 << 30) && (page_size & (page_size - 1)) == 0, DLB_ERR_UNSUPPORTED,
                "%s: page size %lld must be a power of two from 16 on", what, (long long)page_size);
  DLB_CHECK_ARG(num_pages >= 1 && max_pages >= 1, DLB_ERR_BAD_ARG, "%s: empty cache or table", what);
  DLB_CHECK_ARG(num_pages < (1LL << 31) && !too_long(max_pages, page_size) && tokens * hq < (1LL << 31) &&
                    batch <= 65535 && hkv * ((hq / hkv + 15) / 16) <= 65535,
                DLB_ERR_TOO_LARGE, "%s: sizes past 31 bits", what);
  if (softcap > FLT_MAX) softcap = 0.f;       // as good as none
  // the maximum is taken before the scale is applied
  DLB_CHECK_ARG(sm_scale > 0.f, DLB_ERR_BAD_ARG, "%s: sm_scale must be positive", what);
  DLB_CHECK_ARG(!(softcap > 0.f) || sm_scale / softcap <= 1e8f, DLB_ERR_UNSUPPORTED, "%s: soft-cap %g too small", what, (double)softcap);
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

// CTAs to a (row tile, kv head), for `pairs` of them with up to `blocks` blocks.  In microseconds a CTA takes about 4 for everything
// but its blocks, 2 more for a join, and for a block 0.6 alone on its SM and 0.9 beside another.  Clusters only where all of
// them run at once: behind a first wave each costs about 10 more.  Measured with 1 / 2 / 4 / 8 (us, 4 heads to a kv head, 128 columns):
//    64 pairs of 65 blocks  58.3 / 40.1 / 30.8 / 44.5      128 pairs of 65 blocks  58.8 / 48.2 / 56.8 / 83.1
//    64 pairs of  4 blocks  10.1 / 15.2 / 13.4 / 26.0      256 pairs of 65 blocks  71.0 / 71.7 / 89.7 / 140.7
//   640 pairs of 17 blocks  76.7 / 120 / 168 / 323        1024 pairs of 1 to 64     132 / 202 / 286 / 499
static int pick_packed_cluster(int64_t pairs, int64_t blocks) {
  int best = 1;
  int64_t best_cost = INT64_MAX;
  for (int c = 1; c <= MAX_CLUSTER && (c == 1 || pairs * c <= cluster_slots(c)); c *= 2) {
    const int64_t cost = (blocks + c - 1) / c * (2 * pairs * c <= cluster_slots(c) ? 6 : 9) + 40 + (c > 1 ? 20 : 0);
    if (cost < best_cost) {
      best = c;
      best_cost = cost;
    }
  }
  return best;
}

// `tokens` is how many tokens of a sequence (or group) there are at most, or on average: where their rows fit half a tile, tiles
// are half as high, which leaves room for a third K and V buffer.
static void set_shape(PackedParams& p, int64_t tokens, int64_t hq, int64_t hkv, int width, float sm_scale, float softcap, int dtype) {
  p.hq = (int)hq;
  p.hkv = (int)hkv;
  p.group = (int)(hq / hkv);
  p.tile_tokens = (tokens * p.group <= pa::BM / 2 ? pa::BM / 2 : pa::BM) / p.group;
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
                           max_pages, sm_scale, softcap, dtype, width);
  if (rc != DLB_OK) return rc;
  DLB_CHECK_ARG(window >= 0 && sinks >= 0 && max_q_len >= 0, DLB_ERR_BAD_ARG, "sink_attention: negative window, sinks or length");
  if (batch == 0 || total_q_tokens == 0 || max_q_len == 0) return DLB_OK;
  DLB_CHECK_ARG(q && k_cache && v_cache && out && block_table && q_start_loc && q_seq_len && kv_seq_len, DLB_ERR_BAD_ARG,
                "sink_attention: null pointer");
  rc = check_rows("sink_attention", q, out, q_stride_t, q_stride_h, o_stride_t, o_stride_h);
  if (rc != DLB_OK) return rc;
  const int win = (int)(window < INT_MAX ? window : INT_MAX), snk = (int)(sinks < INT_MAX ? sinks : INT_MAX);
  const int64_t most_keys = (int64_t)win + snk, room = max_pages * page_size;
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
    const int64_t bound = most_keys + 1 < room ? most_keys + 1 : room;
    return launch_cluster_decode(d, k_cache, v_cache, k_stride_page, k_stride_slot, k_stride_head, v_stride_page,
                                 v_stride_slot, v_stride_head, width, bound, dtype, s);
  }
  PackedParams p = {};
  set_shape(p, max_q_len, hq, hkv, width, sm_scale, softcap, dtype);
  p.out = out; p.q_start = q_start_loc; p.q_lens = q_seq_len; p.kv_lens = kv_seq_len; p.block_table = block_table;
  p.o_st = o_stride_t; p.o_sh = o_stride_h; p.bt_stride = bt_stride;
  p.tokens = total_q_tokens;
  p.batch = (int)batch;
  p.page_shift = log2_of(page_size); p.max_pages = (int)max_pages; p.num_pages = (int)num_pages; p.dv = (int)head_dim_v;
  p.table_is_int64 = table_is_int64; p.start_is_int64 = start_is_int64; p.qlens_is_int64 = qlen_is_int64; p.lens_is_int64 = kvlen_is_int64;
  p.window = win; p.sinks = snk; p.status = status;
  const int64_t tiles = total_q_tokens / p.tile_tokens + batch;      // sequences end inside a tile at most once each
  DLB_CHECK_ARG(tiles * hkv * MAX_CLUSTER < (1LL << 31), DLB_ERR_TOO_LARGE, "sink_attention: grid too large");
  p.tiles = (int)tiles;
  const int64_t seen = most_keys + p.tile_tokens < room ? most_keys + p.tile_tokens : room;
  const int64_t likely = batch * ((total_q_tokens / batch + p.tile_tokens - 1) / p.tile_tokens);      // with sequences of one length
  p.cluster = pick_packed_cluster((likely < tiles ? likely : tiles) * hkv, (seen + pa::BN - 1) / pa::BN);
  CUtensorMap tq, tk, tv;
  rc = make_tmap_tokens(&tq, q, head_dim, hq, total_q_tokens, q_stride_h, q_stride_t, p.tile_tokens, p.group);
  if (rc != DLB_OK) return rc;
  const int box = (int)(page_size < pa::BN ? page_size : pa::BN);
  p.k_whole = box == pa::BN && head_dim == width;
  rc = make_tmap_rows(&tk, k_cache, head_dim, hkv, page_size, num_pages, k_stride_page, k_stride_slot, k_stride_head, box, p.k_whole);
  if (rc != DLB_OK) return rc;
  p.v_whole = box == pa::BN && head_dim_v == width;
  rc = make_tmap_rows(&tv, v_cache, head_dim_v, hkv, page_size, num_pages, v_stride_page, v_stride_slot, v_stride_head, box, p.v_whole);
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
    int64_t cluster, float sm_scale, float softcap, int dtype, int32_t* status, void* stream) {
  DLB_NVTX("dlb_shared_prefix_attention");
  using namespace dlb;
  int width = 0;
  int rc = check_attention("shared_prefix_attention", batch, batch, hq, hkv, head_dim, head_dim_v, page_size, num_pages,
                           max_pages < prefix_max_pages ? max_pages : prefix_max_pages, sm_scale, softcap, dtype, width);
  if (rc != DLB_OK) return rc;
  DLB_CHECK_ARG(groups >= 1 && groups <= 65535 && !too_long(prefix_max_pages, page_size) && !too_long(max_pages, page_size),
                DLB_ERR_TOO_LARGE, "shared_prefix_attention: number of groups or length of a table out of range");
  DLB_CHECK_ARG(chunk >= 64 && chunk % 64 == 0 && chunk < (1LL << 31), DLB_ERR_BAD_ARG,
                "shared_prefix_attention: chunk %lld must be a multiple of 64", (long long)chunk);
  DLB_CHECK_ARG(cluster == 1 || cluster == 2 || cluster == 4 || cluster == 8, DLB_ERR_BAD_ARG,
                "shared_prefix_attention: cluster %lld must be 1, 2, 4 or 8", (long long)cluster);
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
  set_shape(p, (batch + groups - 1) / groups, hq, hkv, width, sm_scale, softcap, dtype);
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
  p.cluster = (int)cluster;
  DLB_CHECK_ARG(tiles * hkv * splits * cluster < (1LL << 31), DLB_ERR_TOO_LARGE, "shared_prefix_attention: grid too large");
  p.tiles = (int)tiles;
  CUtensorMap tq, tk, tv;
  rc = make_tmap_tokens(&tq, q, head_dim, hq, batch, q_stride_h, q_stride_t, p.tile_tokens, p.group);
  if (rc != DLB_OK) return rc;
  const int box = (int)(page_size < pa::BN ? page_size : pa::BN);
  p.k_whole = box == pa::BN && head_dim == width;
  rc = make_tmap_rows(&tk, k_cache, head_dim, hkv, page_size, num_pages, k_stride_page, k_stride_slot, k_stride_head, box, p.k_whole);
  if (rc != DLB_OK) return rc;
  p.v_whole = box == pa::BN && head_dim_v == width;
  rc = make_tmap_rows(&tv, v_cache, head_dim_v, hkv, page_size, num_pages, v_stride_page, v_stride_slot, v_stride_head, box, p.v_whole);
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
