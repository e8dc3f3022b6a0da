// Eviction from the 8-bit cache by accumulated attention weight.
//
// kv8_select_kernel, one CTA per (sequence, kv head): the weight of the last token that stays, by three histograms over 11, 11 and
// 10 bits of an order-preserving image of the weights, then the kept positions in order: each warp has a stretch of the sequence,
// counts what lies above and at the threshold, and writes behind the warps before it; of equal weights the earlier stay. The first
// and last tokens that stay in any case are outside the search.
// kv8_move_kernel, one CTA per (block of the result, kv head, keys or values): gathers its rows. The block's scale is the largest of
// those that its rows come from, so a code moves by a power of two: bit for bit where the scales agree.
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

__global__ void __launch_bounds__(SELECT_THREADS) kv8_select_kernel(const EvictArgs p) {
  __shared__ uint32_t hist[2048];
  __shared__ uint32_t s_warp[32];
  __shared__ uint32_t s_digit, s_above;
  griddep_wait();
  griddep_launch();
  const int h = blockIdx.x, b = blockIdx.y;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = evict_len(p, b), budget = p.e.budget;
  if (tid == 0) {
    if (h == 0) p.e.lens[b] = min(n, budget);
    if (p.s.ctx[b] > n) atomicCAS(p.s.status, 0, ST_BAD_ARGS);
  }
  const float* w = p.e.w + b * p.e.w_seq + h * p.e.w_head;
  int* kept = p.e.kept + (long(b) * p.c.Hkv + h) * budget;
  float* w_out = p.e.w_out + (long(b) * p.c.Hkv + h) * budget;
  if (n <= budget) {
    for (int i = tid; i < budget; i += SELECT_THREADS) {
      kept[i] = i < n ? i : -1;
      w_out[i] = i < n ? w[i] : 0.f;
    }
    return;
  }
  const int first = p.e.first, last = p.e.last, mid = n - first - last, want = budget - first - last;
  for (int i = tid; i < first; i += SELECT_THREADS) { kept[i] = i; w_out[i] = w[i]; }
  for (int i = tid; i < last; i += SELECT_THREADS) { kept[budget - last + i] = n - last + i; w_out[budget - last + i] = w[n - last + i]; }
  if (want <= 0) return;
  w += first;
  // threshold: the want-th largest image; `above`: how many are larger
  uint32_t prefix = 0, left = want;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11;
    const uint32_t mask = pass == 0 ? 0u : (pass == 1 ? 0xffe00000u : 0xfffffc00u);
    for (int i = tid; i < 2048; i += SELECT_THREADS) hist[i] = 0;
    __syncthreads();
    for (int i0 = 0; i0 < mid; i0 += SELECT_THREADS) {
      const int i = i0 + tid;
      const uint32_t u = i < mid ? image(w[i]) : 0u;
      const bool in = i < mid && (u & mask) == prefix;
      const uint32_t d = (u >> shift) & ((1u << bits) - 1);
      // many tokens that got nothing: whole warps with one digit count at once
      const uint32_t act = __ballot_sync(0xffffffffu, in);
      if (act) {
        const uint32_t d0 = __shfl_sync(0xffffffffu, d, __ffs(act) - 1);
        if (__all_sync(0xffffffffu, !in || d == d0)) {
          if (lane == 0) atomicAdd(&hist[d0], __popc(act));
        } else if (in) {
          atomicAdd(&hist[d], 1u);
        }
      }
    }
    __syncthreads();
    // digits from the top: the one in which the left-th lies
    uint32_t a = hist[2047 - 2 * tid], c2 = hist[2046 - 2 * tid], sum = a + c2;
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
    __syncthreads();
    prefix |= s_digit << shift;
    left -= s_above;
    __syncthreads();
  }
  // `left` of those equal to the threshold stay, the earliest
  const int per = ((mid + 31) / 32 + 31) / 32 * 32, lo = min(mid, warp * per), hi = min(mid, lo + per);
  uint32_t gt = 0, eq = 0;
  for (int i0 = lo; i0 < hi; i0 += 32) {
    const int i = i0 + lane;
    const uint32_t u = i < hi ? image(w[i]) : 0u;
    gt += __popc(__ballot_sync(0xffffffffu, i < hi && u > prefix));
    eq += __popc(__ballot_sync(0xffffffffu, i < hi && u == prefix));
  }
  if (lane == 0) { hist[warp] = gt; hist[32 + warp] = eq; }
  __syncthreads();
  uint32_t gt0 = 0, eq0 = 0;
  for (int i = 0; i < warp; ++i) { gt0 += hist[i]; eq0 += hist[32 + i]; }
  for (int i0 = lo; i0 < hi; i0 += 32) {
    const int i = i0 + lane;
    const float x = i < hi ? w[i] : 0.f;
    const uint32_t u = image(x);
    const uint32_t mg = __ballot_sync(0xffffffffu, i < hi && u > prefix), me = __ballot_sync(0xffffffffu, i < hi && u == prefix);
    const uint32_t below = (1u << lane) - 1;
    const uint32_t e = eq0 + __popc(me & below);
    if (i < hi && (u > prefix || (u == prefix && e < left))) {
      const uint32_t at = first + gt0 + __popc(mg & below) + min(e, left);
      kept[at] = first + i;
      w_out[at] = x;
    }
    gt0 += __popc(mg);
    eq0 += __popc(me);
  }
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
  cudaError_t r = launch_pdl(kv8_select_kernel, dim3(c.Hkv, s.n), dim3(SELECT_THREADS), 0, st, p);
  const int blocks = (e.budget + c.page - 1) / c.page;
  if (r == cudaSuccess) r = launch_pdl(kv8_move_kernel, dim3(unsigned(blocks) * c.Hkv * 2, s.n), dim3(256), 0, st, p);
  if (r != cudaSuccess) kv8_set_error(cudaGetErrorString(r));
  return r != cudaSuccess;
}

}  // namespace lb
