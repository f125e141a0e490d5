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
// HBM-bound, about 4 FLOP per byte.  The keys that a sequence can see are bounded by the window, so a cluster of at most
// 8 CTAs is split enough and no partial result leaves the SMs; that saves the second launch and the workspace which a
// split over an unbounded length needs.  A tile is 64 keys.  One producer lane per box issues TMA tile loads into a
// 3-stage ring; at the ends of a range 16-row boxes fetch only what some key of the range needs, so that 4 sinks cost
// 16 rows and not 64, and pages that hold no visible key are not looked at (a cache that drops tokens behind the
// window may have reused them).  Four consumer warps own 16 keys of a tile each: mma.sync m16n8k16 with the q-heads
// of the kv head as the M rows.
#include <math_constants.h>

#include "cluster_decode.cuh"

namespace dlb {

namespace cd {
constexpr int TILE = 64;
constexpr int CONSUMERS = 4;
constexpr int THREADS = 32 * (CONSUMERS + 1);
constexpr int STAGES = 3;
constexpr int EDGE_ROWS = 16;
constexpr int MAX_CLUSTER = 8;
template <int D> struct Layout {
  static constexpr int HALF_BYTES = TILE * 128;             // one 64-key x 64-column swizzled box
  static constexpr int BOXES = D / 64;
  static constexpr int KV_BYTES = BOXES * HALF_BYTES;
  static constexpr int STAGE_BYTES = 2 * KV_BYTES;
  static constexpr int RING = STAGES * STAGE_BYTES;
  // after the loop the ring holds the warps' results and the CTA's
  static constexpr int RED_FLOATS = CONSUMERS * 16 * (D + 2);
  static constexpr int JOIN_FLOATS = 16 * (D + 2);
  static constexpr int RESULTS = (RED_FLOATS + JOIN_FLOATS) * 4;
  static constexpr int CTRL = RING > RESULTS ? RING : RESULTS;
  static constexpr int SMEM = CTRL + 128 + 1024;            // 1 KiB to align the ring
};
}  // namespace cd

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ float peer_load(uint32_t smem_addr, int rank) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

template <typename T, int D, bool CAP, bool PREFIX>
__global__ void __launch_bounds__(cd::THREADS, 2)
cluster_decode_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                      const __grid_constant__ CUtensorMap edge_k, const __grid_constant__ CUtensorMap edge_v,
                      const __grid_constant__ ClusterDecodeParams p) {
  using namespace cd;
  using L = Layout<D>;
  constexpr int KSTEPS = D / 16;
  constexpr int NT = D / 8;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + L::CTRL);
  uint64_t* empty_bar = full_bar + STAGES;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty_bar + STAGES);
  volatile int* ext_splits = abort_flag + 1;

  const int rank = blockIdx.x, cluster = gridDim.x;
  const int kvh = blockIdx.y % p.hkv;
  const int hblk = blockIdx.y / p.hkv;                       // block of 16 q-heads of the kv head
  const int b = blockIdx.z;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  // ---- the sequence: its row of q, its keys ----
  const int page_size = 1 << p.page_shift;
  int64_t row = b;
  int ctx = load_index(p.kv_lens, b, p.lens_is_int64);
  if (!PREFIX) {
    const int q_len = load_index(p.q_lens, b, p.qlens_is_int64);
    row = load_index(p.q_start, b, p.start_is_int64);
    if (q_len <= 0 || row < 0 || row >= p.tokens) return;    // the whole cluster leaves
    ctx -= q_len - 1;                                        // its first token (there is one)
  }
  ctx = (int)min((int64_t)ctx, (int64_t)p.max_pages << p.page_shift);
  const int lo = (p.window >= 0 && ctx - 1 > p.window) ? ctx - 1 - p.window : 0;
  const int sink_end = min(p.sinks, lo);
  const int base = lo & ~(TILE - 1);
  const int sink_tiles = (sink_end + TILE - 1) / TILE;
  const int tiles = ctx > 0 ? sink_tiles + (ctx - base + TILE - 1) / TILE : 0;
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

  const int rows_valid = min(16, p.group - hblk * 16);       // q-heads of this CTA
  const int head0 = kvh * p.group + hblk * 16;
  float m_run[2] = {-CUDART_INF_F, -CUDART_INF_F};
  float l_run[2] = {0.f, 0.f};
  float oacc[NT][4];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) oacc[t][j] = 0.f;

  if (warp == CONSUMERS) {
    // ------------------------------ producer ------------------------------
    if (lane == 0) {
      tma_prefetch_desc(&tmap_k);
      tma_prefetch_desc(&tmap_v);
      tma_prefetch_desc(&edge_k);
      tma_prefetch_desc(&edge_v);
    }
    // One table entry per lane: `units` pages (or pieces of 64 slots) to a tile, 32 / units tiles to a batch, the next
    // batch under way while this one is used.
    const int unit_shift = min(p.page_shift, 6);
    const int units = TILE >> unit_shift, batch_tiles = 32 / units;
    auto look_up = [&](int t) {
      t += lane / units;
      if (t >= t_hi) return 0;
      int at, from, to;
      tile_keys(t, at, from, to);
      const int tok = at + ((lane % units) << unit_shift);
      if (tok >= to || tok + (1 << unit_shift) <= from) return 0;          // nothing visible here: not looked at
      const int column = tok >> p.page_shift;
      const int page = load_index(p.block_table, (int64_t)b * p.bt_stride + column, p.table_is_int64);
      if (page >= 0 && page < p.num_pages) return page;
      if (kvh == 0 && hblk == 0) report_bad_page(p.status, b, column, page);
      return 0;
    };
    int pages = look_up(t_lo), pages_next = look_up(t_lo + batch_tiles);
    for (int t = t_lo; t < t_hi; ++t) {
      const int i = t - t_lo, in_batch = i % batch_tiles;
      if (i > 0 && in_batch == 0) {
        pages = pages_next;
        pages_next = look_up(t + batch_tiles);
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
  } else {
    // ------------------------------ consumers ------------------------------
    const int r0 = lane >> 2;        // fragment row (q-head) 0..7, second row is r0 + 8
    const int cq = (lane & 3) * 2;   // fragment column pair
    uint32_t qf[KSTEPS][4];
    {
      const T* qb = reinterpret_cast<const T*>(p.q) + row * p.q_st;
#pragma unroll
      for (int ks = 0; ks < KSTEPS; ++ks) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = r0 + (j & 1) * 8;
          const int col = ks * 16 + cq + (j >> 1) * 8;
          uint32_t v = 0;
          if (r < rows_valid && col < p.dk) v = *reinterpret_cast<const uint32_t*>(qb + (int64_t)(head0 + r) * p.q_sh + col);
          qf[ks][j] = v;
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
          n = prefix_splits(p.prefix, load_index(p.prefix.lens, g0 + __ffs(has) - 1, p.prefix.lens_is_int64));
          break;
        }
      }
      if (lane == 0) *ext_splits = n;
    }
    const float scale2 = p.sm_scale * 1.4426950408889634f;
    const float cap_in = CAP ? p.sm_scale / p.softcap : 0.f, cap_out = p.softcap * 1.4426950408889634f;
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

      // ---- S = Q K^T for this warp's 16 keys ----
      float sacc[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int u = 0; u < 4; ++u) sacc[j][u] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KSTEPS; ++ks) {
        const int key = warp * 16 + (mat >> 1) * 8 + mrow;
        const int ch = ks * 2 + (mat & 1);
        const uint32_t addr = kbase + (ch >> 3) * L::HALF_BYTES + key * 128 + (((ch & 7) ^ (key & 7)) << 4);
        uint32_t b00, b01, b10, b11;
        ldmatrix_x4(addr, b00, b01, b10, b11);
        mma_16816<T>(sacc[0], qf[ks], b00, b01);
        mma_16816<T>(sacc[1], qf[ks], b10, b11);
      }

      // ---- scale, soft-cap, mask, running maximum (base-2 domain) ----
      float mx[2] = {-CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          float v = sacc[j][u];
          if (CAP) v = cap_out * tanhf(v * cap_in);
          else v *= scale2;
          if (partly) {
            const int key = key0 + j * 8 + cq + (u & 1);
            v = (key >= from && key < to) ? v : -CUDART_INF_F;
          }
          sacc[j][u] = v;
          mx[u >> 1] = fmaxf(mx[u >> 1], v);
        }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
      }
      float alpha[2];
      bool grew = false;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float m_new = fmaxf(m_run[r], mx[r]);
        alpha[r] = (m_new == -CUDART_INF_F) ? 1.f : fast_exp2(m_run[r] - m_new);
        grew |= (m_new > m_run[r]) && (m_run[r] != -CUDART_INF_F);
        m_run[r] = m_new;
      }
      float psum[2] = {0.f, 0.f};
      uint32_t pf[4];
      {
        float pv[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float mref = m_run[u >> 1];
            const float e = (mref == -CUDART_INF_F) ? 0.f : fast_exp2(sacc[j][u] - mref);
            pv[j][u] = e;
            psum[u >> 1] += e;
          }
        pf[0] = pack_pair<T>(pv[0][0], pv[0][1]);
        pf[1] = pack_pair<T>(pv[0][2], pv[0][3]);
        pf[2] = pack_pair<T>(pv[1][0], pv[1][1]);
        pf[3] = pack_pair<T>(pv[1][2], pv[1][3]);
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) l_run[r] = l_run[r] * alpha[r] + psum[r];
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int tt = 0; tt < NT; ++tt) {
          oacc[tt][0] *= alpha[0];
          oacc[tt][1] *= alpha[0];
          oacc[tt][2] *= alpha[1];
          oacc[tt][3] *= alpha[1];
        }
      }

      // ---- O += P V ----
#pragma unroll
      for (int n = 0; n < D / 16; ++n) {
        const int key = warp * 16 + (mat & 1) * 8 + mrow;
        const int ch = n * 2 + (mat >> 1);
        const uint32_t addr = vbase + (ch >> 3) * L::HALF_BYTES + key * 128 + (((ch & 7) ^ (key & 7)) << 4);
        uint32_t v00, v01, v10, v11;
        ldmatrix_x4_trans(addr, v00, v01, v10, v11);
        mma_16816<T>(oacc[2 * n], pf, v00, v01);
        mma_16816<T>(oacc[2 * n + 1], pf, v10, v11);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty_bar[s]);
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {    // each lane summed its own 4 keys of a row
      l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 1);
      l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 2);
    }
  }

  // ------------------------------ join the warps ------------------------------
  __syncthreads();   // every load has been consumed: the ring can be reused
  float* red_o = reinterpret_cast<float*>(smem);             // [warps][16][D]
  float* red_m = red_o + CONSUMERS * 16 * D;                 // [warps][16]
  float* red_l = red_m + CONSUMERS * 16;
  float* join_o = red_l + CONSUMERS * 16;                    // [16][D], the CTA's result
  float* join_m = join_o + 16 * D;
  float* join_l = join_m + 16;
  if (warp < CONSUMERS) {
    const int r0 = lane >> 2;
    const int cq = (lane & 3) * 2;
#pragma unroll
    for (int tt = 0; tt < NT; ++tt) {
      float2* o0 = reinterpret_cast<float2*>(red_o + (warp * 16 + r0) * D + tt * 8 + cq);
      float2* o1 = reinterpret_cast<float2*>(red_o + (warp * 16 + r0 + 8) * D + tt * 8 + cq);
      *o0 = make_float2(oacc[tt][0], oacc[tt][1]);
      *o1 = make_float2(oacc[tt][2], oacc[tt][3]);
    }
    if ((lane & 3) == 0) {
      red_m[warp * 16 + r0] = m_run[0];
      red_m[warp * 16 + r0 + 8] = m_run[1];
      red_l[warp * 16 + r0] = l_run[0];
      red_l[warp * 16 + r0 + 8] = l_run[1];
    }
  }
  __syncthreads();
  T* out = reinterpret_cast<T*>(p.out) + row * p.o_st;
  for (int idx = threadIdx.x; idx < rows_valid * D; idx += THREADS) {
    const int r = idx / D;
    const int d = idx - r * D;
    float m = -CUDART_INF_F;
#pragma unroll
    for (int w = 0; w < CONSUMERS; ++w) m = fmaxf(m, red_m[w * 16 + r]);
    float acc = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < CONSUMERS; ++w) {
      const float mw = red_m[w * 16 + r];
      const float sc = (mw == -CUDART_INF_F) ? 0.f : fast_exp2(mw - m);
      acc += red_o[(w * 16 + r) * D + d] * sc;
      l += red_l[w * 16 + r] * sc;
    }
    if (!PREFIX && cluster == 1) {
      if (d < p.dv) out[(int64_t)(head0 + r) * p.o_sh + d] = Elem<T>::from_f(l > 0.f ? acc / l : 0.f);
    } else {
      join_o[idx] = acc;
      if (d == 0) {
        join_m[r] = m;
        join_l[r] = l;
      }
    }
  }
  if (!PREFIX && cluster == 1) return;

  // ------------------------------ join the cluster (and the prefix) ------------------------------
  if (cluster > 1) cluster_barrier();
  else __syncthreads();
  const uint32_t addr_o = smem_u32(join_o), addr_m = smem_u32(join_m), addr_l = smem_u32(join_l);
  const int ext = PREFIX ? *ext_splits : 0;
  for (int idx = rank * THREADS + threadIdx.x; idx < rows_valid * D; idx += cluster * THREADS) {
    const int r = idx / D;
    const int d = idx - r * D;
    float m = -CUDART_INF_F;
    for (int c = 0; c < cluster; ++c) m = fmaxf(m, peer_load(addr_m + r * 4, c));
    const int64_t prow = row * p.hq + head0 + r, rows_all = p.tokens * p.hq;
    if constexpr (PREFIX)
      for (int s = 0; s < ext; ++s) m = fmaxf(m, p.prefix.ml[s * rows_all + prow].x);
    float acc = 0.f, l = 0.f;
    for (int c = 0; c < cluster; ++c) {
      const float mc = peer_load(addr_m + r * 4, c);
      const float sc = (mc == -CUDART_INF_F) ? 0.f : fast_exp2(mc - m);
      acc += peer_load(addr_o + idx * 4, c) * sc;
      l += peer_load(addr_l + r * 4, c) * sc;
    }
    if constexpr (PREFIX) {
      for (int s = 0; s < ext; ++s) {
        const float2 ml = p.prefix.ml[s * rows_all + prow];
        const float sc = (ml.x == -CUDART_INF_F) ? 0.f : fast_exp2(ml.x - m);
        acc += p.prefix.o[(s * rows_all + prow) * D + d] * sc;
        l += ml.y * sc;
      }
    }
    if (d < p.dv) out[(int64_t)(head0 + r) * p.o_sh + d] = Elem<T>::from_f(l > 0.f ? acc / l : 0.f);
  }
  if (cluster > 1) cluster_barrier();    // a CTA's shared memory stays until its peers have read it
}

// CTAs to a (sequence, kv head): doubled while the launch leaves SMs without work, down to two tiles a CTA, and up to four
// waves of two CTAs per SM while a CTA keeps eight tiles.
static int pick_cluster(int64_t pairs, int64_t tiles) {
  int c = 1;
  const int64_t slots = 2 * sm_count(current_device());
  while (c < cd::MAX_CLUSTER && ((pairs * c < slots && tiles >= 4 * c) || (pairs * c < 4 * slots && tiles >= 16 * c))) c *= 2;
  return c;
}

template <typename T, int D, bool CAP, bool PREFIX>
static int launch_cluster(const CUtensorMap (&maps)[4], const ClusterDecodeParams& p, int cluster, cudaStream_t stream) {
  auto kern = cluster_decode_kernel<T, D, CAP, PREFIX>;
  constexpr int SMEM = cd::Layout<D>::SMEM;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
  if (e != cudaSuccess) {
    set_last_error("cluster_decode: cannot raise dynamic shared memory: %s", cudaGetErrorString(e));
    return (int)e;
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cluster, p.hkv * ((p.group + 15) / 16), p.batch);
  cfg.blockDim = dim3(cd::THREADS);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kern, maps[0], maps[1], maps[2], maps[3], p);
  if (e != cudaSuccess) {
    set_last_error("cluster_decode: launch failed: %s", cudaGetErrorString(e));
    (void)cudaGetLastError();
    return (int)e;
  }
  return DLB_OK;
}
template <typename T, int D>
static int launch_cluster(const CUtensorMap (&maps)[4], const ClusterDecodeParams& p, int cluster, cudaStream_t stream) {
  const bool cap = p.softcap > 0.f;
  if (p.prefix.o != nullptr)
    return cap ? launch_cluster<T, D, true, true>(maps, p, cluster, stream)
               : launch_cluster<T, D, false, true>(maps, p, cluster, stream);
  return cap ? launch_cluster<T, D, true, false>(maps, p, cluster, stream)
             : launch_cluster<T, D, false, false>(maps, p, cluster, stream);
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
  const int64_t pairs = (int64_t)p.batch * p.hkv * ((p.group + 15) / 16);
  const int cluster = pick_cluster(pairs, (key_bound + cd::TILE - 1) / cd::TILE);
  if (dtype == DLB_DTYPE_BF16)
    return width == 128 ? launch_cluster<__nv_bfloat16, 128>(maps, p, cluster, stream)
                        : launch_cluster<__nv_bfloat16, 64>(maps, p, cluster, stream);
  return width == 128 ? launch_cluster<__half, 128>(maps, p, cluster, stream)
                      : launch_cluster<__half, 64>(maps, p, cluster, stream);
}

}  // namespace dlb
