// Eviction from the 8-bit cache by accumulated attention weight.
//
// kv8_select_kernel, a cluster of 1 to 8 CTAs per (sequence, kv head), each with a stretch of the sequence, order-preserving images
// of its weights in shared memory: the weight of the last token that stays, by three histograms over 11, 11 and 10 bits, summed over
// the cluster through distributed shared memory, then the kept positions in order: each warp counts what lies above and at the
// threshold in its part and writes behind the warps and CTAs before it; of equal weights the earlier stay. The first and last tokens
// that stay in any case are outside the search. It is kept small: a launch fetches its code anew. (4 sequences of 32K tokens and 4
// heads: one CTA each 45 us, weights in registers by unrolled code 75, clusters of eight 63: half of them wait for the others.)
// kv8_move_kernel, one CTA per (block of the result, kv head, keys or values): gathers its rows. The block's scale is the largest of
// those that its rows come from, so a code moves by a power of two: bit for bit where the scales agree. 4 sequences of 32K tokens to
// 4096, 4 heads of 128: selection 25 us (shared-memory atomics), moving 12 us.
#include <cooperative_groups.h>

#include "kv8_dev.cuh"

namespace lb {
namespace {

constexpr int SELECT_THREADS = 1024;

struct EvictArgs {
  Kv8Cache c;
  Kv8Seqs s;
  Kv8Evict e;
};

__device__ __forceinline__ int evict_len(const EvictArgs& p, int b) {
  const int n = int(min(long(max(p.s.ctx[b], 0)), long(p.s.width) * p.c.page));
  return min(n, p.e.w_keys);
}

// larger image = larger weight; NaN above everything
__device__ __forceinline__ uint32_t image(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int HELD = 50 * 1024;        // images in a CTA's shared memory; those of a longer stretch's rest are made again in every pass

__global__ void __launch_bounds__(SELECT_THREADS) kv8_select_kernel(const EvictArgs p, int room) {
  namespace cg = cooperative_groups;
  extern __shared__ uint32_t held[];
  __shared__ __align__(16) uint32_t hist[2048];
  __shared__ uint32_t s_warp[32], s_gt[32], s_eq[32];
  __shared__ uint32_t s_digit, s_above, s_cta[2];
  griddep_wait();
  griddep_launch();
  const cg::cluster_group cl = cg::this_cluster();
  const int n_cta = int(cl.num_blocks()), rank = int(cl.block_rank());
  const int h = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = evict_len(p, b), budget = p.e.budget;
  if (tid == 0 && rank == 0) {
    if (h == 0) p.e.lens[b] = min(n, budget);
    if (p.s.ctx[b] > n) atomicCAS(p.s.status, 0, ST_BAD_ARGS);
  }
  const float* w = p.e.w + b * p.e.w_seq + h * p.e.w_head;
  int* kept = p.e.kept + (long(b) * p.c.Hkv + h) * budget;
  float* w_out = p.e.w_out + (long(b) * p.c.Hkv + h) * budget;
  const int step = n_cta * SELECT_THREADS, me_all = rank * SELECT_THREADS + tid;
  if (n <= budget) {                                        // (the whole cluster)
    for (int i = me_all; i < budget; i += step) {
      kept[i] = i < n ? i : -1;
      w_out[i] = i < n ? w[i] : 0.f;
    }
    return;
  }
  const int first = p.e.first, last = p.e.last, mid = n - first - last, want = budget - first - last;
  for (int i = me_all; i < first; i += step) { kept[i] = i; w_out[i] = w[i]; }
  for (int i = me_all; i < last; i += step) { kept[budget - last + i] = n - last + i; w_out[budget - last + i] = w[n - last + i]; }
  if (want <= 0) return;
  // this CTA's stretch [c0, c1) of the tokens that are searched, and this warp's part of it, [lo, hi)
  const int per = ((mid + n_cta * 32 - 1) / (n_cta * 32) + 31) / 32 * 32;
  const int c0 = int(min(long(mid), long(rank) * 32 * per)), c1 = int(min(long(mid), c0 + 32l * per)), len = c1 - c0;
  const int lo = min(len, warp * per), hi = min(len, lo + per);
  w += first + c0;
  const int n_held = min(len, room);
#pragma unroll 4
  for (int i = tid; i < n_held; i += SELECT_THREADS) held[i] = image(w[i]);
  auto image_of = [&](int i) { return i < n_held ? held[i] : image(w[i]); };
  // threshold: the want-th largest image; `left`: how many equal to it stay
  uint32_t prefix = 0, left = want;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11;
    const uint32_t mask = pass == 0 ? 0u : (pass == 1 ? 0xffe00000u : 0xfffffc00u);
    for (int i = tid; i < 2048; i += SELECT_THREADS) hist[i] = 0;
    __syncthreads();
#pragma unroll 1
    for (int i0 = 0; i0 < len; i0 += SELECT_THREADS) {
      const int i = i0 + tid;
      const uint32_t u = i < len ? image_of(i) : 0u;
      const bool in = i < len && (u & mask) == prefix;
      const uint32_t d = (u >> shift) & ((1u << bits) - 1);
      // many tokens that got nothing: whole warps with one digit count at once
      const uint32_t act = __ballot_sync(0xffffffffu, in);
      if (act == 0) continue;
      const uint32_t d0 = __shfl_sync(0xffffffffu, d, __ffs(act) - 1);
      if (__all_sync(0xffffffffu, !in || d == d0)) {
        if (lane == 0) atomicAdd(&hist[d0], __popc(act));
      } else if (in) {
        atomicAdd(&hist[d], 1u);
      }
    }
    // digits from the top, two to a thread, over the cluster: the digit in which the left-th lies
    cl.sync();
    uint32_t a = 0, c2 = 0;
    for (int r = 0; r < n_cta; ++r) {
      const uint2 x = *reinterpret_cast<const uint2*>(cl.map_shared_rank(hist, r) + 2046 - 2 * tid);
      a += x.y;
      c2 += x.x;
    }
    const uint32_t sum = a + c2;
    uint32_t inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    if (warp == 0) {
      uint32_t v = s_warp[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
      }
      s_warp[lane] = v;
    }
    __syncthreads();
    const uint32_t before = inc - sum + (warp ? s_warp[warp - 1] : 0u);
    if (before < left && left <= before + a) { s_digit = 2047 - 2 * tid; s_above = before; }
    else if (before + a < left && left <= before + sum) { s_digit = 2046 - 2 * tid; s_above = before + a; }
    cl.sync();                                              // nobody reads this histogram any more
    prefix |= s_digit << shift;
    left -= s_above;
  }
  // counts above and at the threshold of every warp, and of the warps before this one
  uint32_t gt = 0, eq = 0;
#pragma unroll 2
  for (int i0 = lo; i0 < hi; i0 += 32) {
    const int i = i0 + lane;
    const uint32_t u = i < hi ? image_of(i) : 0u;
    gt += __popc(__ballot_sync(0xffffffffu, i < hi && u > prefix));
    eq += __popc(__ballot_sync(0xffffffffu, i < hi && u == prefix));
  }
  if (lane == 0) { s_gt[warp] = gt; s_eq[warp] = eq; }
  __syncthreads();
  uint32_t gt0 = lane < warp ? s_gt[lane] : 0u, eq0 = lane < warp ? s_eq[lane] : 0u;
  gt0 = __reduce_add_sync(0xffffffffu, gt0);
  eq0 = __reduce_add_sync(0xffffffffu, eq0);
  if (tid == SELECT_THREADS - 1) { s_cta[0] = gt0 + s_gt[31]; s_cta[1] = eq0 + s_eq[31]; }
  cl.sync();
  for (int r = 0; r < rank; ++r) {
    const uint32_t* x = cl.map_shared_rank(s_cta, r);
    gt0 += x[0];
    eq0 += x[1];
  }
#pragma unroll 2
  for (int i0 = lo; i0 < hi; i0 += 32) {
    const int i = i0 + lane;
    const uint32_t u = i < hi ? image_of(i) : 0u;
    const uint32_t mg = __ballot_sync(0xffffffffu, i < hi && u > prefix), me = __ballot_sync(0xffffffffu, i < hi && u == prefix);
    const uint32_t below = (1u << lane) - 1, e = eq0 + __popc(me & below);
    if (i < hi && (u > prefix || (u == prefix && e < left))) {
      const uint32_t at = first + gt0 + __popc(mg & below) + min(e, left);
      kept[at] = first + c0 + i;
      w_out[at] = w[i];
    }
    gt0 += __popc(mg);
    eq0 += __popc(me);
  }
  cl.sync();                                                // counts are read until here
}

__global__ void __launch_bounds__(256) kv8_move_kernel(const EvictArgs p) {
  __shared__ float s_scale[64];
  __shared__ long s_src[64];
  griddep_wait();
  griddep_launch();
  const Kv8Cache& c = p.c;
  const int b = blockIdx.y, h = (blockIdx.x >> 1) % c.Hkv, j = (blockIdx.x >> 1) / c.Hkv;
  const bool val = blockIdx.x & 1;
  const int len = min(evict_len(p, b), p.e.budget);
  const int rows = min(c.page, len - j * c.page);
  if (rows <= 0) return;
  const int dst = p.e.dst[b * p.e.ld_dst + j];
  if (unsigned(dst) >= unsigned(c.n_blocks)) {
    if (threadIdx.x == 0) atomicCAS(p.s.status, 0, ST_BAD_ARGS);
    return;
  }
  const int D = val ? c.dv : c.dk, per = D / 16;
  uint8_t* codes = val ? c.v : c.k;
  float* scales = val ? c.v_scale : c.k_scale;
  if (threadIdx.x < rows) {
    const int t = p.e.kept[(long(b) * c.Hkv + h) * p.e.budget + j * c.page + threadIdx.x];
    const int blk = p.s.table[b * p.s.ld_table + t / c.page];
    const bool ok = unsigned(blk) < unsigned(c.n_blocks);
    if (!ok) atomicCAS(p.s.status, 0, ST_BAD_ARGS);
    s_src[threadIdx.x] = ok ? ((long(blk) * c.Hkv + h) * c.page + t % c.page) * D : -1;
    s_scale[threadIdx.x] = ok ? scales[long(blk) * c.Hkv + h] : 0.f;
  }
  __syncthreads();
  float now = 0.f;
  for (int i = 0; i < rows; ++i) now = fmaxf(now, s_scale[i]);
  const float inv = kv8_inverse(now);
  const long unit = long(dst) * c.Hkv + h;
  for (int at = threadIdx.x; at < c.page * per; at += 256) {
    const int r = at / per, col = (at % per) * 16;
    uint4 u = make_uint4(0u, 0u, 0u, 0u);
    if (r < rows && s_src[r] >= 0) {
      u = *reinterpret_cast<const uint4*>(codes + s_src[r] + col);
      if (s_scale[r] != now || now == 0.f) {
        const float by = s_scale[r] * inv;
        uint32_t* w = &u.x;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 x = __half22float2(e4m3x2_to_half2(w[k])), y = __half22float2(e4m3x2_to_half2(w[k] >> 16));
          w[k] = e4m3x2(x.x * by, x.y * by) | e4m3x2(y.x * by, y.y * by) << 16;
        }
      }
    }
    *reinterpret_cast<uint4*>(codes + (unit * c.page + r) * D + col) = u;
  }
  if (threadIdx.x == 0) scales[unit] = now;
}

}  // namespace

int kv8_evict_launch(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Evict& e, cudaStream_t st) {
  if (s.n <= 0) return 0;
  const EvictArgs p{c, s, e};
  const long most = long(s.width) * c.page < e.w_keys ? long(s.width) * c.page : e.w_keys;
  // CTAs of a sequence and head: from 4096 tokens each, while the SMs have room for all (clusters of eight find it harder)
  int n_cta = 1;
  while (n_cta < 8 && most > long(n_cta) * 4096 && long(n_cta) * 2 * c.Hkv * s.n <= (n_cta < 4 ? 148 : 64)) n_cta *= 2;
  const long stretch = (most + n_cta - 1) / n_cta + 1024;
  const int room = stretch < HELD ? int(stretch) : HELD;
  static DeviceOnce once;
  cudaError_t r = once.shared_memory(reinterpret_cast<const void*>(kv8_select_kernel), HELD * 4);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(n_cta, c.Hkv, s.n);
  cfg.blockDim = dim3(SELECT_THREADS);
  cfg.dynamicSmemBytes = size_t(room) * 4;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = n_cta;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  if (r == cudaSuccess) r = cudaLaunchKernelEx(&cfg, kv8_select_kernel, p, room);
  const int blocks = (e.budget + c.page - 1) / c.page;
  if (r == cudaSuccess) r = launch_pdl(kv8_move_kernel, dim3(unsigned(blocks) * c.Hkv * 2, s.n), dim3(256), 0, st, p);
  if (r != cudaSuccess) kv8_set_error(cudaGetErrorString(r));
  return r != cudaSuccess;
}

}  // namespace lb
