// Single-token attention split over a thread-block cluster (cluster_decode.cu), as its callers see it.
#pragma once
#include <limits.h>
#include <math_constants.h>

#include <atomic>

#include "attention.cuh"

namespace dlb {

constexpr int MAX_CLUSTER = 8;

// CTAs of two to an SM that run at the same time in clusters of c: a cluster stays inside a GPC, so that larger ones leave
// slots empty (296, 296, 284 and 264 on the B200 that was asked).
static inline int64_t cluster_slots(int c) {
  const int64_t all = 2 * sm_count(current_device());
  return c <= 2 ? all : c == 4 ? all * 95 / 100 : all * 88 / 100;
}

// Partial results of the shared prefixes, one row per (token, q-head): unnormalised output, then the reference maximum
// (base-2 domain) and the sum that go with it.
struct PrefixPartials {
  float* o;                    // [splits, tokens * hq, D]
  float2* ml;                  // [splits, tokens * hq]
  const void* lens;            // [groups] tokens of each prefix
  const void* group_start;     // [groups + 1] first token (row of q) of each group
  int groups, lens_is_int64, start_is_int64;
  int max_len;                 // tokens the prefix table has room for
  int chunk;                   // tokens per split, a multiple of 64
};

struct ClusterDecodeParams {
  const void* q;               // [tokens, hq, dk]
  void* out;                   // [tokens, hq, dv]
  const void* block_table;     // [batch, max_pages]
  const void* kv_lens;         // [batch]
  const void* q_start;         // [batch] row of each sequence, with q_lens (none where it is 0); null: row b
  const void* q_lens;
  int64_t q_st, q_sh, o_st, o_sh, bt_stride;
  int64_t tokens;
  int batch, hq, hkv, group, dk, dv;
  int page_shift, max_pages, num_pages;
  int table_is_int64, lens_is_int64, start_is_int64, qlens_is_int64;
  int window, sinks;           // window < 0: every key
  float sm_scale, softcap;     // softcap <= 0: none
  int* status;
  PrefixPartials prefix;       // o == null: none
};

// Entry i of an index array; 64-bit ones are kept inside 32 bits, where a page, a row or a length out there stays out of range.
__device__ __forceinline__ int clamped_index(const void* p, int64_t i, int is64) {
  if (!is64) return reinterpret_cast<const int32_t*>(p)[i];
  return (int)max((int64_t)INT_MIN, min((int64_t)INT_MAX, reinterpret_cast<const int64_t*>(p)[i]));
}

// Records a page that does not exist where a visible token should be.
__device__ __forceinline__ void report_bad_page(int* status, int row, int column, int page) {
  if (status != nullptr && atomicCAS(status, DLB_DEV_OK, DLB_DEV_BAD_PAGE) == DLB_DEV_OK) {
    status[1] = row;
    status[2] = column;
    status[3] = page;
  }
}

// Splits of a prefix of `len` tokens (as many as the table has room for).
__device__ __forceinline__ int prefix_splits(const PrefixPartials& p, int len) {
  return (int)(((uint32_t)max(min(len, p.max_len), 0) + (uint32_t)p.chunk - 1) / (uint32_t)p.chunk);    // the sum may pass 2^31
}

// Rows [start, start + n) of group g, kept inside the rows that exist.
__device__ __forceinline__ void group_rows(const PrefixPartials& p, int64_t tokens, int g, int& start, int& n) {
  const int64_t lo = p.start_is_int64 ? reinterpret_cast<const int64_t*>(p.group_start)[g]
                                      : reinterpret_cast<const int32_t*>(p.group_start)[g];
  const int64_t hi = p.start_is_int64 ? reinterpret_cast<const int64_t*>(p.group_start)[g + 1]
                                      : reinterpret_cast<const int32_t*>(p.group_start)[g + 1];
  const int64_t a = max((int64_t)0, min(lo, tokens));
  start = (int)a;
  n = (int)max((int64_t)0, min(hi, tokens) - a);
}

// cap * tanh(x) in the base-2 domain from one exponential and one reciprocal: tanh(x) = 1 - 2 / (1 + e^2x).  Off by 2^-22 of
// the cap, so for scores that come near it; `in` = 2 log2(e) sm_scale / cap, `out` = cap log2(e).
__device__ __forceinline__ float soft_cap(float s, float in, float out) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + fast_exp2(s * in)));
  return fmaf(-2.f * out, r, out);
}
// The same without the special-function unit: tanh(x) = x P(x^2), P interpolated at the Chebyshev nodes, off by 2^-21 of the
// score with 32-bit coefficients (a score is a sum of up to 128 rounded products), for |x| <= 1 (7 terms) or 1/4 (3).  Two
// scores at a time; x = sm_scale / cap goes into the argument of the long form and, once for a row, into the coefficients
// of the short one.
__device__ __forceinline__ uint64_t soft_cap_below(uint64_t s, uint64_t x, uint64_t out) {     // out = sm_scale log2(e)
  constexpr float P[7] = {0.99999995f, -0.33332828f, 0.13325076f, -0.05345165f, 0.02027971f, -0.00619432f, 0.00103803f};
  const uint64_t u1 = mul_f2(s, x), u = mul_f2(u1, u1);
  uint64_t p = pack_f2(P[6], P[6]);
#pragma unroll
  for (int i = 5; i >= 0; --i) p = fma_f2(p, u, pack_f2(P[i], P[i]));
  return mul_f2(mul_f2(s, out), p);
}
struct SoftCapShort {
  uint64_t c0, c1, c2;
  __device__ __forceinline__ SoftCapShort(float x, float out) {
    const float a = 0.99999958f * out, b = -0.33321896f * out * (x * x), c = 0.12841433f * out * (x * x) * (x * x);
    c0 = pack_f2(a, a);
    c1 = pack_f2(b, b);
    c2 = pack_f2(c, c);
  }
  __device__ __forceinline__ uint64_t operator()(uint64_t s) const {
    const uint64_t u = mul_f2(s, s);
    return mul_f2(s, fma_f2(fma_f2(c2, u, c1), u, c0));
  }
};

// Two scores of any size: the small ones by the polynomial, since the other way is off by 2^-22 of the cap, however large that is.
__device__ __forceinline__ void soft_cap_any(float& a, float& b, const SoftCapShort& low, float x, float in, float out) {
  float la, lb;
  unpack_f2(low(pack_f2(a, b)), la, lb);
  a = fabsf(a * x) <= 0.25f ? la : soft_cap(a, in, out);
  b = fabsf(b * x) <= 0.25f ? lb : soft_cap(b, in, out);
}

// Behind a wait that gave up: waits, again with a limit, for what is still under way to a ring of barriers (copies, commits of
// matrix instructions), so that nothing lands in the shared memory of a CTA that has left.  `used` uses of the ring have begun.
__device__ __forceinline__ void settle_ring(uint64_t* ring, int stages, int used) {
  for (int s = 0; s < stages && s < used; ++s) {
    const uint32_t last = (uint32_t)((used - 1 - s) / stages) & 1;
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(&ring[s], last) && globaltimer_ns() - t0 < DLB_WAIT_BUDGET_NS) {
    }
  }
}

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_address(uint32_t smem_addr, int rank) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr), "r"(rank));
  return at;
}
__device__ __forceinline__ float peer_load(uint32_t at) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float4 peer_load4(uint32_t at) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}
// One running result (m, l, four columns) takes in another.
struct Joined {
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  __device__ __forceinline__ void add(float pm, float pl, const float4& po) {
    if (pl == 0.f) return;                                  // a piece without keys
    const float top = fmaxf(m, pm);
    const float a = m == -CUDART_INF_F ? 0.f : fast_exp2(m - top), b = fast_exp2(pm - top);
    m = top;
    l = l * a + pl * b;
    o.x = o.x * a + po.x * b;
    o.y = o.y * a + po.y * b;
    o.z = o.z * a + po.z * b;
    o.w = o.w * a + po.w * b;
  }
};

// Columns d .. d + 3 of an output row of dv, rounded once; a row that saw no key is zero (a sum that is no number stays one).
template <typename T> __device__ __forceinline__ void store_joined(T* out_row, int d, int dv, const Joined& j) {
  if (d >= dv) return;
  const float inv = j.l == 0.f ? 0.f : 1.f / j.l;
  typename Elem<T>::T2 v[2] = {Elem<T>::from_f2(j.o.x * inv, j.o.y * inv), Elem<T>::from_f2(j.o.z * inv, j.o.w * inv)};
  *reinterpret_cast<uint2*>(out_row + d) = *reinterpret_cast<const uint2*>(v);
}

// A launch that says so may start once every CTA of the launch before it has begun and called let_next_start (or ended); it
// sees that launch's results behind wait_for_previous.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Launch in clusters of `cluster` CTAs along x; `early` as above.  The kernel's shared memory is raised once per device.
template <auto KERN, typename... Args>
static int launch_in_clusters(const char* what, dim3 grid, int threads, int smem, int cluster, bool early,
                              cudaStream_t stream, const Args&... args) {
  static std::atomic<uint64_t> raised{0};
  const int dev = current_device();
  cudaError_t e = cudaSuccess;
  if (dev >= 64 || !(raised.load(std::memory_order_relaxed) >> dev & 1)) {
    e = cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess && dev < 64) raised.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  if (e == cudaSuccess) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = early ? 2 : 1;
    e = cudaLaunchKernelEx(&cfg, KERN, args...);
  }
  if (e != cudaSuccess) {
    set_last_error("%s: launch failed: %s", what, cudaGetErrorString(e));
    (void)cudaGetLastError();
    return (int)e;
  }
  return DLB_OK;
}

// `width` is the tile width (64 or 128); key_bound the keys that one sequence can see at most.
int launch_cluster_decode(const ClusterDecodeParams& p, const void* k_cache, const void* v_cache, int64_t k_stride_page,
                          int64_t k_stride_slot, int64_t k_stride_head, int64_t v_stride_page, int64_t v_stride_slot,
                          int64_t v_stride_head, int width, int64_t key_bound, int dtype, cudaStream_t stream);

}  // namespace dlb
