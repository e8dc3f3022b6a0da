// Writing the 8-bit key/value cache.
//
// kv8_append: one CTA per (block that gets tokens, kv head, keys or values). The rows that join the block stay in registers
// between the search for the largest magnitude and the encoding, so every input byte is read once:
//     s' = max(s, 2^(floor(log2 amax) - 7)),   code = e4m3(x / s'),   older codes = e4m3(code * s / s')
// A block whose first cell is written begins anew (s = 0, other cells become zero). Blocks belong to one sequence, so a CTA has
// its block to itself and nothing depends on the order of CTAs. 8192 tokens, 4 heads of 128: 9.7 us = 2.6 TB/s, where lengths,
// table and rows are dependent reads; a token for each of 16 sequences is bound by its launch.
#include "kv8_dev.cuh"

namespace lb {
namespace {

constexpr int APPEND_THREADS = 256;

struct AppendArgs {
  Kv8Cache c;
  Kv8Seqs s;
  Kv8Append a;
  int vec;                         // input rows start on 16 bytes
};

__device__ __forceinline__ uint4 load_row8(const __nv_bfloat16* p, bool vec) {
  if (vec) return *reinterpret_cast<const uint4*>(p);
  uint4 u;
  const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
  u.x = h[0] | uint32_t(h[1]) << 16; u.y = h[2] | uint32_t(h[3]) << 16;
  u.z = h[4] | uint32_t(h[5]) << 16; u.w = h[6] | uint32_t(h[7]) << 16;
  return u;
}

// largest finite magnitude of two bf16 (as a bf16 pattern in 16 bits: magnitudes order as whole numbers); NaN is left out,
// infinities count as the largest finite value
__device__ __forceinline__ uint32_t mag2(uint32_t w) {
  uint32_t lo = w & 0x7fffu, hi = (w >> 16) & 0x7fffu;
  lo = lo > 0x7f80u ? 0u : min(lo, 0x7f7fu);
  hi = hi > 0x7f80u ? 0u : min(hi, 0x7f7fu);
  return max(lo, hi);
}
__device__ __forceinline__ uint32_t encode2(uint32_t w, float inv) {
  float lo = __uint_as_float(w << 16), hi = __uint_as_float(w & 0xffff0000u);
  if (fabsf(lo) > KV8_MOST) lo = copysignf(KV8_MOST, lo);      // infinities (NaN compares false and stays)
  if (fabsf(hi) > KV8_MOST) hi = copysignf(KV8_MOST, hi);
  return e4m3x2(lo * inv, hi * inv);
}

template <int VPT>      // vectors of eight values that a thread holds
__global__ void __launch_bounds__(APPEND_THREADS) kv8_append_kernel(const AppendArgs p) {
  __shared__ uint32_t s_max[APPEND_THREADS / 32];
  griddep_wait();
  griddep_launch();
  const Kv8Cache& c = p.c;
  const int b = blockIdx.y, h = (blockIdx.x >> 1) % c.Hkv, j = (blockIdx.x >> 1) / c.Hkv;
  const bool val = blockIdx.x & 1;
  const int row0 = p.s.cu[b], n = p.s.cu[b + 1] - row0;
  const int len = max(p.s.ctx[b], 0), ctx = int(min(long(len), long(p.s.width) * c.page));
  const int first = max(len - n, 0);                         // position of the first new token
  if (n <= 0 || first >= ctx) return;
  const int col = first / c.page + j;
  const int lo = max(first, col * c.page), hi = min(ctx, (col + 1) * c.page);
  if (lo >= hi) return;
  if (row0 < 0 || long(row0) + n > p.s.T || n > p.s.max_new) {
    if (threadIdx.x == 0) atomicCAS(p.s.status, 0, ST_BAD_ARGS);
    return;
  }
  const int blk = p.s.table[b * p.s.ld_table + col];
  const int D = val ? c.dv : c.dk, per = D / 8;
  const long tok = val ? p.a.v_tok : p.a.k_tok;
  const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(val ? p.a.v : p.a.k) + (val ? p.a.v_head : p.a.k_head) * h +
                             (row0 + (lo - (len - n))) * tok;
  const int nvec = (hi - lo) * per;
  uint4 x[VPT];                                             // on their way while the table answers
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int at = threadIdx.x + i * APPEND_THREADS;
    if (at < nvec) {
      x[i] = load_row8(src + (at / per) * tok + (at % per) * 8, p.vec);
    }
  }
  if (unsigned(blk) >= unsigned(c.n_blocks)) {
    if (threadIdx.x == 0) atomicCAS(p.s.status, 0, ST_BAD_ARGS);
    return;
  }
  const long unit = long(blk) * c.Hkv + h;
  uint8_t* codes = (val ? c.v : c.k) + unit * c.page * D;
  float* scale = (val ? c.v_scale : c.k_scale) + unit;
  const float old = lo == col * c.page ? 0.f : *scale;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (threadIdx.x + i * APPEND_THREADS < nvec) m = max(max(m, max(mag2(x[i].x), mag2(x[i].y))), max(mag2(x[i].z), mag2(x[i].w)));
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
  __syncthreads();                                          // (every thread has read the old scale, too)
#pragma unroll
  for (int i = 0; i < APPEND_THREADS / 32; ++i) m = max(m, s_max[i]);
  const float now = fmaxf(old, kv8_scale_of(__uint_as_float(m << 16)));
  const float inv = kv8_inverse(now);
  uint8_t* dst = codes + (lo - col * c.page) * D;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int at = threadIdx.x + i * APPEND_THREADS;
    if (at < nvec) {
      uint2 u;
      u.x = encode2(x[i].x, inv) | encode2(x[i].y, inv) << 16;
      u.y = encode2(x[i].z, inv) | encode2(x[i].w, inv) << 16;
      *reinterpret_cast<uint2*>(dst + long(at) * 8) = u;
    }
  }
  if (threadIdx.x == 0) *scale = now;
  if (now == old && now != 0.f) return;
  // the block's other cells: zero in a block that begins, rounded to the new scale in one whose scale grew
  const bool begun = lo == col * c.page;
  const float by = old * inv;
  const int v0 = (lo - col * c.page) * per, v1 = v0 + nvec;
  for (int at = threadIdx.x; at < c.page * per; at += APPEND_THREADS) {
    if (at >= v0 && at < v1) continue;
    uint2* cell = reinterpret_cast<uint2*>(codes + long(at) * 8);
    uint2 u = make_uint2(0u, 0u);
    if (!begun) {
      const uint2 w = *cell;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = __half22float2(e4m3x2_to_half2((k < 2 ? w.x : w.y) >> (16 * (k & 1))));
        (k < 2 ? u.x : u.y) |= e4m3x2(f.x * by, f.y * by) << (16 * (k & 1));
      }
    }
    *cell = u;
  }
}

}  // namespace

static thread_local char g_kv8_err[256];
const char* kv8_last_error() { return g_kv8_err; }
void kv8_set_error(const char* what) { snprintf(g_kv8_err, sizeof(g_kv8_err), "%s", what); }

int kv8_append_launch(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Append& a, cudaStream_t st) {
  if (s.n <= 0 || s.max_new <= 0 || s.T <= 0) return 0;
  AppendArgs p{c, s, a, 0};
  p.vec = ((reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v)) & 15) == 0 &&
          (a.k_tok | a.k_head | a.v_tok | a.v_head) % 8 == 0;
  // blocks that `max_new` tokens can touch
  const long cols = (long(s.max_new) + c.page - 2) / c.page + 1;
  const dim3 grid(unsigned(cols * c.Hkv * 2), unsigned(s.n));
  const int most = (c.page < s.max_new ? c.page : s.max_new) * (c.dk > c.dv ? c.dk : c.dv) / 8;
  cudaError_t e;
  if (most <= APPEND_THREADS) e = launch_pdl(kv8_append_kernel<1>, grid, dim3(APPEND_THREADS), 0, st, p);
  else if (most <= 4 * APPEND_THREADS) e = launch_pdl(kv8_append_kernel<4>, grid, dim3(APPEND_THREADS), 0, st, p);
  else e = launch_pdl(kv8_append_kernel<8>, grid, dim3(APPEND_THREADS), 0, st, p);
  if (e != cudaSuccess) kv8_set_error(cudaGetErrorString(e));
  return e != cudaSuccess;
}

}  // namespace lb
