// Single-token attention over a paged cache, split over a thread-block cluster: the keys of one (sequence, kv head) are
// cut into as many pieces as the cluster has CTAs, and the pieces are joined through distributed shared memory in the
// same launch.  Two users: attention with a sliding window and sinks, and the own tokens of sequences that share a
// prefix, whose partial results over the prefix join in the same place.
//
// Math: the query at position p sees the keys j <= p with j >= p - window or j < sinks, in two ranges
//     [0, min(sinks, lo))  and  [lo, p],   lo = max(0, p - window);
// scores q.k * sm_scale (optional tanh soft-cap), softmax with a running maximum and sum in 32 bits, P rounded to the
// cache's 16-bit type for the matrix instructions (half a step of 2^-8 for bf16, 2^-11 for fp16, on weights that are then
// averaged), pieces joined by 2^(m_piece - m).
//
// HBM-bound, about 4 FLOP per byte.  At most 8 CTAs share the keys of a (sequence, kv head), and no partial result leaves the
// SMs; that saves the second launch and the workspace which a split over the whole GPU needs.  It is split enough for windows
// and own tokens of some thousand keys, and for batches that fill the SMs; one sequence over 131072 keys takes 178 us with one
// kv head of 128 columns, where paged_decode.cu takes 123, and 199 with eight (195).  A tile is 64 keys.  One producer lane per box issues TMA tile loads into a
// 2-stage ring; at the ends of a range 16-row boxes fetch only what some key of the range needs, so that 4 sinks cost
// 16 rows and not 64, and pages that hold no visible key are not looked at (a cache that drops tokens behind the
// window may have reused them).  Four consumer warps own 16 keys of a tile each and compute S^T = K Q^T and O^T += V^T P
// with mma.sync m16n8k16: keys (columns of V) are the 16 rows, eight q-heads of the kv head the 8 columns, so that 4 or 8
// heads do not leave three quarters or half of the rows empty.  Against q-heads as rows this halves instructions and
// accumulators, which lets three CTAs with two stages share an SM in place of two with three: 64 sequences with a window of
// 4096, 8 kv heads, 128 columns: 202 -> 182 us (5.9 TB/s); 256 sequences of 16 to 512 own tokens and 8 pieces of a prefix:
// 98 -> 58 us.
#include <math_constants.h>

#include "cluster_decode.cuh"

namespace dlb {

namespace cd {
constexpr int TILE = 64;
constexpr int CONSUMERS = 4;
constexpr int THREADS = 32 * (CONSUMERS + 1);
constexpr int STAGES = 2;
constexpr int EDGE_ROWS = 16;
constexpr float RESCALE_THRESHOLD = 8.0f;                   // log2 units: P stays below 2^8, well inside fp16
template <int D, int NH> struct Layout {
  static constexpr int HEADS = 8 * NH;                      // q-heads to a CTA
  static constexpr int HALF_BYTES = TILE * 128;             // one 64-key x 64-column swizzled box
  static constexpr int BOXES = D / 64;
  static constexpr int KV_BYTES = BOXES * HALF_BYTES;
  static constexpr int STAGE_BYTES = 2 * KV_BYTES;
  static constexpr int RING = STAGES * STAGE_BYTES;
  // after the loop the ring holds the warps' results and the CTA's, rows of PITCH floats (4 more than D, so that the lanes
  // of a store, 8 columns of 4 heads, fall on 32 banks)
  static constexpr int PITCH = D + 4;
  static constexpr int RESULTS = (CONSUMERS + 1) * HEADS * (PITCH + 2) * 4;
  static constexpr int CTRL = RING > RESULTS ? RING : RESULTS;
  static constexpr int SMEM = CTRL + 128 + 1024;            // 1 KiB to align the ring
};
}  // namespace cd

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

template <typename T, int D, int NH, bool CAP, bool PREFIX>
__global__ void __launch_bounds__(cd::THREADS, NH == 1 ? 3 : 2)
cluster_decode_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                      const __grid_constant__ CUtensorMap edge_k, const __grid_constant__ CUtensorMap edge_v,
                      const __grid_constant__ ClusterDecodeParams p) {
  using namespace cd;
  using L = Layout<D, NH>;
  constexpr int KSTEPS = D / 16;
  constexpr int MT = D / 16;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + L::CTRL);
  uint64_t* empty_bar = full_bar + STAGES;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty_bar + STAGES);
  volatile int* ext_splits = abort_flag + 1;
  volatile int* loaded = abort_flag + 2;                     // tiles that were asked for

  const int rank = blockIdx.x, cluster = gridDim.x;
  const int kvh = blockIdx.y % p.hkv;
  const int hblk = blockIdx.y / p.hkv;                       // block of q-heads of the kv head
  const int b = blockIdx.z;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (warp == CONSUMERS && lane == 0) {
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
    tma_prefetch_desc(&edge_k);
    tma_prefetch_desc(&edge_v);
  }

  // ---- the sequence: its row of q, its keys ----
  const int page_size = 1 << p.page_shift;
  int64_t row = b;
  int64_t len = clamped_index(p.kv_lens, b, p.lens_is_int64);
  if (!PREFIX) {
    const int q_len = clamped_index(p.q_lens, b, p.qlens_is_int64);
    row = clamped_index(p.q_start, b, p.start_is_int64);
    if (q_len <= 0 || row < 0 || row >= p.tokens) return;    // the whole cluster leaves
    len -= q_len - 1;                                        // its first token (there is one)
  }
  // the keys that are there; a query past them keeps its position
  const int ctx = (int)max((int64_t)0, min(len, (int64_t)p.max_pages << p.page_shift));
  const int lo = p.window >= 0 ? (int)max((int64_t)0, min(len - 1 - p.window, (int64_t)ctx)) : 0;
  const int sink_end = min(p.sinks, lo);
  const int base = lo & ~(TILE - 1);
  const int sink_tiles = (sink_end + TILE - 1) / TILE;
  const int tiles = sink_tiles + (ctx > lo ? (ctx - base + TILE - 1) / TILE : 0);
  const int t_lo = (int)((int64_t)tiles * rank / cluster), t_hi = (int)((int64_t)tiles * (rank + 1) / cluster);
  // tile t starts at key `at` and the keys [from, to) count
  auto tile_keys = [&](int t, int& at, int& from, int& to) {
    const bool sink = t < sink_tiles;
    at = sink ? t * TILE : base + (t - sink_tiles) * TILE;
    from = sink ? 0 : lo;
    to = sink ? sink_end : ctx;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], CONSUMERS);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();

  const int rows_valid = min(L::HEADS, p.group - hblk * L::HEADS);   // q-heads of this CTA
  const int head0 = kvh * p.group + hblk * L::HEADS;
  // a thread's heads: 8 n + (lane & 3) * 2 and the next
  float m_run[NH][2], l_run[NH][2];
  float oacc[NH][MT][4];
#pragma unroll
  for (int n = 0; n < NH; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      m_run[n][e] = -CUDART_INF_F;
      l_run[n][e] = 0.f;
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) oacc[n][t][j] = 0.f;
  }

  if (warp == CONSUMERS) {
    // ------------------------------ producer ------------------------------
    // One table entry per lane: `units` pages (or pieces of 64 slots) to a tile, 32 / units tiles to a batch.  The next batch's
    // entries are asked for when this one's come into use, and looked at only then.
    const int unit_shift = min(p.page_shift, 6);
    const int units = TILE >> unit_shift, batch_tiles = 32 / units;
    auto lane_token = [&](int t, bool& wanted) {             // first key of this lane's piece of the batch from tile t on
      t += lane / units;
      int at, from, to;
      tile_keys(t, at, from, to);
      const int tok = at + ((lane % units) << unit_shift);
      wanted = t < t_hi && tok < to && tok + (1 << unit_shift) > from;     // else nothing visible here: not looked at
      return tok;
    };
    auto entry = [&](int t) {
      bool wanted;
      const int64_t column = lane_token(t, wanted) >> p.page_shift;
      return wanted ? clamped_index(p.block_table, (int64_t)b * p.bt_stride + column, p.table_is_int64) : 0;
    };
    int pages = 0, pages_next = entry(t_lo), asked = 0;
    for (int t = t_lo; t < t_hi; ++t) {
      const int i = t - t_lo, in_batch = i % batch_tiles;
      if (in_batch == 0) {
        pages = pages_next;
        pages_next = entry(t + batch_tiles);
        if (pages < 0 || pages >= p.num_pages) {
          bool wanted;
          const int column = lane_token(t, wanted) >> p.page_shift;
          if (kvh == 0 && hblk == 0) report_bad_page(p.status, b, column, pages);
          pages = 0;
        }
      }
      const int s = i % STAGES;
      const uint32_t ph = (i / STAGES) & 1;
      int at, from, to;
      tile_keys(t, at, from, to);
      const bool edge = at < from || at + TILE > to;
      const int box_shift = edge ? 4 : unit_shift;
      const int tok = at + (lane << box_shift);
      const bool mine = lane < (TILE >> box_shift) && tok < to && tok + (1 << box_shift) > from;
      const int boxes = __popc(__ballot_sync(0xffffffffu, mine));
      int ok = 1;
      if (lane == 0) {
        ok = mbar_wait(&empty_bar[s], ph ^ 1, abort_flag, p.status, 41, t) ? 1 : 0;
        if (ok) mbar_arrive_expect_tx(&full_bar[s], (uint32_t)((boxes << box_shift) * 128 * L::BOXES * 2));
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) break;
      asked = i + 1;
      const int page = __shfl_sync(0xffffffffu, pages, in_batch * units + (min(lane << box_shift, TILE - 1) >> unit_shift));
      if (mine) {
        uint8_t* kdst = smem + s * L::STAGE_BYTES + (lane << box_shift) * 128;
        const CUtensorMap* mk = edge ? &edge_k : &tmap_k;
        const CUtensorMap* mv = edge ? &edge_v : &tmap_v;
        const int slot = tok & (page_size - 1);
#pragma unroll
        for (int h = 0; h < L::BOXES; ++h) {
          tma_load_4d(kdst + h * L::HALF_BYTES, mk, &full_bar[s], h * 64, kvh, slot, page);
          tma_load_4d(kdst + L::KV_BYTES + h * L::HALF_BYTES, mv, &full_bar[s], h * 64, kvh, slot, page);
        }
      }
    }
    if (lane == 0) *loaded = asked;
  } else {
    // ------------------------------ consumers ------------------------------
    // Q^T as the B operand: head lane / 4 (of each block of 8), columns (lane & 3) * 2 of every 8
    uint32_t qf[NH][KSTEPS][2];
    {
      const T* qb = reinterpret_cast<const T*>(p.q) + row * p.q_st;
#pragma unroll
      for (int n = 0; n < NH; ++n) {
        const int r = n * 8 + (lane >> 2);
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ++ks) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int col = ks * 16 + (lane & 3) * 2 + j * 8;
            uint32_t v = 0;
            if (r < rows_valid && col < p.dk) v = *reinterpret_cast<const uint32_t*>(qb + (int64_t)(head0 + r) * p.q_sh + col);
            qf[n][ks][j] = v;
          }
        }
      }
    }
    if (PREFIX && warp == 0) {
      // the splits of the prefix of this row's group (the first group that has it; none: no prefix)
      int n = 0;
      for (int g0 = 0; g0 < p.prefix.groups; g0 += 32) {
        int start = 0, rows = 0;
        if (g0 + lane < p.prefix.groups) group_rows(p.prefix, p.tokens, g0 + lane, start, rows);
        const uint32_t has = __ballot_sync(0xffffffffu, b >= start && b < start + rows);
        if (has != 0) {
          n = prefix_splits(p.prefix, clamped_index(p.prefix.lens, g0 + __ffs(has) - 1, p.prefix.lens_is_int64));
          break;
        }
      }
      if (lane == 0) *ext_splits = n;
    }
    const float scale2 = p.sm_scale * 1.4426950408889634f;
    const float cap_in = CAP ? 2.f * 1.4426950408889634f * p.sm_scale / p.softcap : 0.f, cap_out = p.softcap * 1.4426950408889634f,
                cap_x = CAP ? p.sm_scale / p.softcap : 0.f;
    const SoftCapShort cap_short(cap_x, scale2);
    const int mat = lane >> 3;      // ldmatrix: which 8x8 matrix this lane addresses
    const int mrow = lane & 7;

    for (int t = t_lo; t < t_hi; ++t) {
      const int i = t - t_lo, s = i % STAGES;
      const uint32_t ph = (i / STAGES) & 1;
      bool ok = mbar_wait(&full_bar[s], ph, abort_flag, p.status, 42, t);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const uint32_t kbase = smem_u32(smem + s * L::STAGE_BYTES);
      const uint32_t vbase = kbase + L::KV_BYTES;
      int at, from, to;
      tile_keys(t, at, from, to);
      const int key0 = at + warp * 16;                       // this warp's 16 keys
      const bool partly = key0 < from || key0 + 16 > to;
      if (partly) {
        // V rows that do not count are zeroed: 0 x (whatever an old tile or a reused page left there) may be NaN
        for (int c = lane; c < 16 * (D / 8); c += 32) {
          const int key = key0 + c / (D / 8);
          if (key < from || key >= to) {
            const int chunk = c % (D / 8), r = warp * 16 + c / (D / 8);
            *reinterpret_cast<uint4*>(smem + s * L::STAGE_BYTES + L::KV_BYTES + (chunk >> 3) * L::HALF_BYTES + r * 128 +
                                      (((chunk & 7) ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
          }
        }
        fence_proxy_async_smem();                            // before the copy engine writes this stage again
        __syncwarp();
      }

      // ---- S^T = K Q^T: this warp's 16 keys by 8 NH heads ----
      float sacc[NH][4];
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int u = 0; u < 4; ++u) sacc[n][u] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KSTEPS; ++ks) {
        const int key = warp * 16 + (mat & 1) * 8 + mrow;
        const int ch = ks * 2 + (mat >> 1);
        uint32_t a[4];
        ldmatrix_x4(kbase + (ch >> 3) * L::HALF_BYTES + key * 128 + (((ch & 7) ^ (key & 7)) << 4), a[0], a[1], a[2], a[3]);
#pragma unroll
        for (int n = 0; n < NH; ++n) mma_16816<T>(sacc[n], a, qf[n][ks][0], qf[n][ks][1]);
      }

      // ---- scale, soft-cap, mask (base-2 domain); the reference maximum is raised when a score passes it by 2^8 ----
      bool grow = false;
#pragma unroll
      for (int n = 0; n < NH; ++n) {
        if (CAP) {
          soft_cap_any(sacc[n][0], sacc[n][1], cap_short, cap_x, cap_in, cap_out);
          soft_cap_any(sacc[n][2], sacc[n][3], cap_short, cap_x, cap_in, cap_out);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          float v = CAP ? sacc[n][u] : sacc[n][u] * scale2;
          if (partly) {
            const int key = key0 + (lane >> 2) + (u >> 1) * 8;
            v = (key >= from && key < to) ? v : -CUDART_INF_F;
          }
          sacc[n][u] = v;
          // m_run -inf: any score that is not -inf itself
          grow |= v > m_run[n][u & 1] + RESCALE_THRESHOLD;
        }
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int n = 0; n < NH; ++n) {
          float alpha[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(sacc[n][e], sacc[n][e + 2]);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            mx = fmaxf(mx, m_run[n][e]);
            alpha[e] = m_run[n][e] == -CUDART_INF_F ? 0.f : fast_exp2(m_run[n][e] - mx);
            m_run[n][e] = mx;
            l_run[n][e] *= alpha[e];
          }
#pragma unroll
          for (int tt = 0; tt < MT; ++tt) {
            oacc[n][tt][0] *= alpha[0];
            oacc[n][tt][1] *= alpha[1];
            oacc[n][tt][2] *= alpha[0];
            oacc[n][tt][3] *= alpha[1];
          }
        }
      }
      uint32_t pf[NH][2];
#pragma unroll
      for (int n = 0; n < NH; ++n) {
        float e[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float mref = m_run[n][u & 1];                  // -inf: no score so far but -inf, or one that is no number
          e[u] = fast_exp2(mref == -CUDART_INF_F ? sacc[n][u] : sacc[n][u] - mref);
          l_run[n][u & 1] += e[u];
        }
        pf[n][0] = transpose_8x8(pack_pair<T>(e[0], e[1]));
        pf[n][1] = transpose_8x8(pack_pair<T>(e[2], e[3]));
      }

      // ---- O^T += V^T P ----
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int key = warp * 16 + (mat >> 1) * 8 + mrow;
        const int ch = m * 2 + (mat & 1);
        uint32_t a[4];
        ldmatrix_x4_trans(vbase + (ch >> 3) * L::HALF_BYTES + key * 128 + (((ch & 7) ^ (key & 7)) << 4), a[0], a[1], a[2],
                          a[3]);
#pragma unroll
        for (int n = 0; n < NH; ++n) mma_16816<T>(oacc[n][m], a, pf[n][0], pf[n][1]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty_bar[s]);
    }
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)    // each lane summed its own keys
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l_run[n][e] += __shfl_xor_sync(0xffffffffu, l_run[n][e], o);
  }

  // ------------------------------ join the warps ------------------------------
  __syncthreads();   // every load has been consumed: the ring can be reused
  if (*abort_flag) {
    if (threadIdx.x == 0) settle_ring(full_bar, STAGES, *loaded);
    __syncthreads();
  }
  constexpr int H = L::HEADS, PITCH = L::PITCH, QUADS = D / 4;
  float* red_o = reinterpret_cast<float*>(smem);             // [warps + 1][H][PITCH], the last one the CTA's
  float* red_m = red_o + (CONSUMERS + 1) * H * PITCH;        // [warps + 1][H]
  float* red_l = red_m + (CONSUMERS + 1) * H;
  if (warp < CONSUMERS) {
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      const int h = n * 8 + (lane & 3) * 2;
      float* o = red_o + (warp * H + h) * PITCH + (lane >> 2);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        o[m * 16] = oacc[n][m][0];
        o[PITCH + m * 16] = oacc[n][m][1];
        o[m * 16 + 8] = oacc[n][m][2];
        o[PITCH + m * 16 + 8] = oacc[n][m][3];
      }
      if (lane < 4) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          red_m[warp * H + h + e] = m_run[n][e];
          red_l[warp * H + h + e] = l_run[n][e];
        }
      }
    }
  }
  __syncthreads();
  T* out = reinterpret_cast<T*>(p.out) + row * p.o_st;
  for (int idx = threadIdx.x; idx < rows_valid * QUADS; idx += THREADS) {
    const int r = idx / QUADS, d = idx % QUADS * 4;
    Joined j;
#pragma unroll
    for (int w = 0; w < CONSUMERS; ++w)
      j.add(red_m[w * H + r], red_l[w * H + r], *reinterpret_cast<const float4*>(red_o + (w * H + r) * PITCH + d));
    if (!PREFIX && cluster == 1) {
      store_joined<T>(out + (int64_t)(head0 + r) * p.o_sh, d, p.dv, j);
    } else {
      *reinterpret_cast<float4*>(red_o + (CONSUMERS * H + r) * PITCH + d) = j.o;
      if (d == 0) {
        red_m[CONSUMERS * H + r] = j.m;
        red_l[CONSUMERS * H + r] = j.l;
      }
    }
  }
  if (!PREFIX && cluster == 1) return;

  // ------------------------------ join the cluster (and the prefix) ------------------------------
  if (cluster > 1) cluster_barrier();
  else __syncthreads();
  const uint32_t at_o = smem_u32(red_o + CONSUMERS * H * PITCH), at_m = smem_u32(red_m + CONSUMERS * H),
                 at_l = smem_u32(red_l + CONSUMERS * H);
  // the own tokens are through; the launch with the prefix's partial results may still have been under way
  if (PREFIX) wait_for_previous();
  const int ext = PREFIX ? *ext_splits : 0;
  // Eight lanes take eight quads of a row; where this CTA has few of them, two or four such groups of lanes share their
  // pieces.  Four loads of a lane are under way together; the CTAs of the cluster share the quads.
  constexpr int OCTS = QUADS / 8, GROUPS = 4 * (CONSUMERS + 1);
  const int g_lo = rows_valid * OCTS * rank / cluster, g_hi = rows_valid * OCTS * (rank + 1) / cluster;
  const int parts_shift = (g_hi - g_lo) * 4 <= GROUPS ? 2 : (g_hi - g_lo) * 2 <= GROUPS ? 1 : 0;
  const int parts = 1 << parts_shift, part = (lane >> 3) & (parts - 1);
  const int64_t rows_all = p.tokens * p.hq;
  for (int g0 = g_lo; g0 < g_hi; g0 += GROUPS >> parts_shift) {
    const int g = g0 + ((int)(threadIdx.x >> 3) >> parts_shift);
    const int r = min(g, g_hi - 1) / OCTS, d = (g % OCTS * 8 + (lane & 7)) * 4;
    Joined j;
    for (int c0 = part; c0 < cluster; c0 += 4 * parts) {
      float m[4], l[4];
      float4 o[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int c = min(c0 + u * parts, cluster - 1);
        m[u] = peer_load(peer_address(at_m + r * 4, c));
        l[u] = peer_load(peer_address(at_l + r * 4, c));
        o[u] = peer_load4(peer_address(at_o + (r * PITCH + d) * 4, c));
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (c0 + u * parts < cluster) j.add(m[u], l[u], o[u]);
    }
    if constexpr (PREFIX) {
      const int64_t prow = row * p.hq + head0 + r;
      for (int s = part; s < ext; s += 4 * parts) {
        float2 ml[4];
        float4 o[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int64_t k = min(s + u * parts, ext - 1) * rows_all + prow;
          ml[u] = p.prefix.ml[k];
          o[u] = *reinterpret_cast<const float4*>(p.prefix.o + k * D + d);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (s + u * parts < ext) j.add(ml[u].x, ml[u].y, o[u]);
      }
    }
    for (int o = 8; o < 8 * parts; o <<= 1)
      j.add(__shfl_xor_sync(0xffffffffu, j.m, o), __shfl_xor_sync(0xffffffffu, j.l, o),
            make_float4(__shfl_xor_sync(0xffffffffu, j.o.x, o), __shfl_xor_sync(0xffffffffu, j.o.y, o),
                        __shfl_xor_sync(0xffffffffu, j.o.z, o), __shfl_xor_sync(0xffffffffu, j.o.w, o)));
    if (part == 0 && g < g_hi) store_joined<T>(out + (int64_t)(head0 + r) * p.o_sh, d, p.dv, j);
  }
  if (cluster > 1) cluster_barrier();    // a CTA's shared memory stays until its peers have read it
}

// CTAs to a (sequence, kv head), by the shortest sum over the waves: in tenths of a microsecond a CTA takes 40 for everything but
// its tiles, 25 more for a join, and for a tile 10 alone on its SM, 13 beside another CTA, 22 where three share the memory.
// Measured with 1 / 2 / 4 / 8 (us, tiles of 64 keys x 128 columns, 17 and 65 of them):
//    32 pairs 26.6 / 18.5 / 16.4 / 16.4        64 pairs 71.6 / 49.2 / 40.9 / 49.2       (65)
//   128 pairs 32.7 / 26.7 / 34.8 / 41.0       128 pairs 79.8 / 63.5 / 69.7 / 75.8       (65)
//   256 pairs 38.9 / 49.2 / 53.2 / 71.6       512 pairs 200.7 / 188.4 / 188.4 / 215.0   (65)
static int pick_cluster(int64_t pairs, int64_t tiles, int resident) {
  int best = 1;
  int64_t best_cost = INT64_MAX;
  for (int c = 1; c <= MAX_CLUSTER; c *= 2) {
    const int64_t slots = cluster_slots(c) * resident / 2, ctas = pairs * c, waves = (ctas + slots - 1) / slots;
    const int64_t sms = sm_count(current_device());
    const int64_t tile = waves > 1 || ctas > 2 * sms ? 22 : ctas > sms ? 13 : 10;
    const int64_t cost = waves * ((tiles + c - 1) / c * tile + 40 + (c > 1 ? 25 : 0));
    if (cost < best_cost) {
      best = c;
      best_cost = cost;
    }
  }
  return best;
}

template <typename T, int D, int NH, bool CAP, bool PREFIX>
static int launch_cluster(const CUtensorMap (&maps)[4], const ClusterDecodeParams& p, int cluster, cudaStream_t stream) {
  return launch_in_clusters<cluster_decode_kernel<T, D, NH, CAP, PREFIX>>(
      "cluster_decode", dim3(cluster, p.hkv * ((p.group + 8 * NH - 1) / (8 * NH)), p.batch), cd::THREADS,
      cd::Layout<D, NH>::SMEM, cluster, PREFIX, stream, maps[0], maps[1], maps[2], maps[3], p);
}
template <typename T, int D, int NH>
static int launch_cluster(const CUtensorMap (&maps)[4], const ClusterDecodeParams& p, int cluster, cudaStream_t stream) {
  const bool cap = p.softcap > 0.f;
  if (p.prefix.o != nullptr)
    return cap ? launch_cluster<T, D, NH, true, true>(maps, p, cluster, stream)
               : launch_cluster<T, D, NH, false, true>(maps, p, cluster, stream);
  return cap ? launch_cluster<T, D, NH, true, false>(maps, p, cluster, stream)
             : launch_cluster<T, D, NH, false, false>(maps, p, cluster, stream);
}
template <typename T>
static int launch_cluster(const CUtensorMap (&maps)[4], const ClusterDecodeParams& p, int width, int64_t key_bound,
                          cudaStream_t stream) {
  // up to 8 heads to a kv head fill one block of the B operand; with more a CTA takes 16
  const bool narrow = p.group <= 8;
  const int64_t pairs = (int64_t)p.batch * p.hkv * (narrow ? 1 : (p.group + 15) / 16);
  const int cluster = pick_cluster(pairs, (key_bound + cd::TILE - 1) / cd::TILE, narrow ? 3 : 2);
  if (narrow)
    return width == 128 ? launch_cluster<T, 128, 1>(maps, p, cluster, stream) : launch_cluster<T, 64, 1>(maps, p, cluster, stream);
  return width == 128 ? launch_cluster<T, 128, 2>(maps, p, cluster, stream) : launch_cluster<T, 64, 2>(maps, p, cluster, stream);
}

int launch_cluster_decode(const ClusterDecodeParams& p, const void* k_cache, const void* v_cache, int64_t k_stride_page,
                          int64_t k_stride_slot, int64_t k_stride_head, int64_t v_stride_page, int64_t v_stride_slot,
                          int64_t v_stride_head, int width, int64_t key_bound, int dtype, cudaStream_t stream) {
  const int page = 1 << p.page_shift, full = page < cd::TILE ? page : cd::TILE;
  CUtensorMap maps[4];
  for (int i = 0; i < 4; ++i) {
    const bool k = i % 2 == 0;
    if (i >= 2 && full == cd::EDGE_ROWS) {
      maps[i] = maps[i - 2];
      continue;
    }
    const int rc = make_tmap_cache(&maps[i], k ? k_cache : v_cache, k ? p.dk : p.dv, p.hkv, page, p.num_pages,
                                   k ? k_stride_page : v_stride_page, k ? k_stride_slot : v_stride_slot,
                                   k ? k_stride_head : v_stride_head, i < 2 ? full : cd::EDGE_ROWS);
    if (rc != DLB_OK) return rc;
  }
  return dtype == DLB_DTYPE_BF16 ? launch_cluster<__nv_bfloat16>(maps, p, width, key_bound, stream)
                                 : launch_cluster<__half>(maps, p, width, key_bound, stream);
}

}  // namespace dlb
