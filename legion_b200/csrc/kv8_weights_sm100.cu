// Sums of attention weights per key of the 8-bit cache, for eviction: w[key] += sum over rows and query heads of
// exp(score - lse), with the log-sum-exp of every row and head from the attention itself.
//
// The scores once more, as in the decode kernel: S^T[128 keys, rows] = K . Q^T on tcgen05 with the codes as they are and queries as
// two e4m3 terms side by side in the N dimension. A thread has a key and adds up its columns, so nothing crosses threads and the
// sums do not depend on any order but the rows' own; every key belongs to one CTA, which adds to it once per tile of RN rows.
// Keys and scales are read once per tile of rows: a decode step (up to 16 heads of a kv head) is bound by the keys' bytes, an
// observed window of rows by 64 exponentials per key and tile.
#include "kv8_dev.cuh"
#include "tmap.cuh"

namespace lb {
namespace {

struct WeightArgs {
  Kv8Cache c;
  Kv8Seqs s;
  Kv8Attn a;
  int observe, per;               // last rows of a sequence that count (0: all); key tiles of a CTA
  float scale_log2, cap_k;
  float* w; long w_seq, w_head; int w_keys;
};

template <int KH, int RN>
struct WCfg {
  static constexpr int NS = 2 * RN;
  static constexpr int K_BYTES = KH * 16384, ST = 96 * 1024 / K_BYTES;      // 6 or 3 stages: two CTAs fit an SM
  static constexpr int Q_BYTES = KH * NS * 128;
  static constexpr int TAIL = 2048;
  static constexpr int SMEM = ST * K_BYTES + Q_BYTES + TAIL + 1024;
  static constexpr int TMEM_COLS = 2 * NS < 32 ? 32 : 2 * NS;
  static_assert(SMEM <= 227 * 1024 && TMEM_COLS <= 256, "sizes");
};

template <int BAR, int N>
__device__ __forceinline__ void named_sync() {
  asm volatile("bar.sync %0, %1;" ::"n"(BAR), "n"(N) : "memory");
}

template <int KH, int RN, bool CAP>
__global__ void __launch_bounds__(320, KH == 1 ? 2 : 1) kv8_weights_kernel(const __grid_constant__ CUtensorMap tmK, const WeightArgs p) {
  using C = WCfg<KH, RN>;
  constexpr int BKV = 128, NS = C::NS, ST = C::ST;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* k_s = smem;
  uint8_t* q_s = k_s + ST * C::K_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(q_s + C::Q_BYTES);
  uint64_t* k_full = bars;         // [6]
  uint64_t* k_empty = bars + 6;    // [6]
  uint64_t* s_full = bars + 12;    // [2]
  uint64_t* s_empty = bars + 14;   // [2]
  uint64_t* q_full = bars + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 17);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint32_t* s_max = reinterpret_cast<uint32_t*>(bars + 18);      // [8]
  float* s_lse = reinterpret_cast<float*>(bars + 24);            // [RN]
  int* s_pos = reinterpret_cast<int*>(s_lse + 64);               // [RN]

  const Kv8Cache& c = p.c;
  const int G = p.a.Hq / c.Hkv;
  const int kvh = blockIdx.x, split = blockIdx.y, seq = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  griddep_wait();
  griddep_launch();
  const int q0 = p.s.cu[seq], n_new = p.s.cu[seq + 1] - q0;
  if (n_new <= 0) return;
  const int ctx = int(min(long(max(p.s.ctx[seq], 0)), long(p.s.width) * c.page));
  if (q0 < 0 || long(q0) + n_new > p.s.T || n_new > p.s.max_new || ctx > p.w_keys) {
    if (threadIdx.x == 0) atomicCAS(p.s.status, 0, ST_BAD_ARGS);
    return;
  }
  const int first = p.observe > 0 ? max(0, n_new - p.observe) : 0;      // first row that counts
  const int rows = (n_new - first) * G, n_rt = (rows + RN - 1) / RN;
  const int base = ctx - n_new + first;                                 // its position
  const int tile0 = split * p.per, tile1 = split == int(gridDim.y) - 1 ? (ctx + BKV - 1) / BKV : min((ctx + BKV - 1) / BKV, tile0 + p.per);
  // tiles of this CTA that rows of tile rt see: [from, to)
  auto range = [&](int rt, int& from, int& to) {
    const int a = base + rt * RN / G, b = base + (min(rows, (rt + 1) * RN) - 1) / G;
    const int lo = p.a.window > 0 ? max(0, a - p.a.window + 1) : 0, hi = min(ctx, b + 1);
    from = max(tile0, lo / BKV);
    to = min(tile1, (hi + BKV - 1) / BKV);
  };
  if (tile0 >= tile1) return;

  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], 128);
    }
    mbar_init(q_full, 256);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int* bt = p.s.table + seq * p.s.ld_table;
  auto fail = [&](int code) { *abort_flag = 1; atomicCAS(p.s.status, 0, code | SITE_DECODE_ATTN); return false; };

  if (warp == 9) {
    const int ppb = BKV / c.page;
    bool ok = true;
    int it = 0;
    for (int rt = 0; ok && rt < n_rt; ++rt) {
      int from, to;
      range(rt, from, to);
      int pg_reg = 0;
      const int tiles_per_fill = 32 / ppb;                  // (an empty range runs no tile)
      for (int tile = from; ok && tile < to; ++tile, ++it) {
        const int at = (tile - from) % tiles_per_fill;
        if (at == 0) {
          const long page = long(tile) * ppb + lane;
          pg_reg = page * c.page < ctx ? bt[page] : c.n_blocks;
          if (unsigned(pg_reg) > unsigned(c.n_blocks)) pg_reg = c.n_blocks;      // (reads as zeros; recorded with the scales)
        }
        const int st = it % ST;
        if (it >= ST && !__all_sync(0xffffffffu, mbar_wait(&k_empty[st], ((it / ST) - 1) & 1, abort_flag))) {
          if (lane == 0) fail(ST_TIMEOUT_EMPTY);
          ok = false;
          break;
        }
        if (lane == 0) mbar_expect_tx(&k_full[st], C::K_BYTES);
        for (int g = 0; g < ppb; ++g) {
          const int pg = __shfl_sync(0xffffffffu, pg_reg, at * ppb + g);
          if (lane == 0)
            for (int h = 0; h < KH; ++h)
              tma_load_2d(k_s + st * C::K_BYTES + h * 16384 + g * c.page * 128, &tmK, &k_full[st], h * 128, (pg * c.Hkv + kvh) * c.page);
        }
      }
    }
  } else if (warp == 8) {
    if (lane == 0) {
      constexpr uint32_t idesc = umma_idesc(128, NS, 0, 0, 0, 0);
      const uint64_t dk = umma_desc_k_sw128(smem_u32(k_s)), dq = umma_desc_k_sw128(smem_u32(q_s));
      bool ok = true;
      int it = 0, staged = 0;
      for (int rt = 0; ok && rt < n_rt; ++rt) {
        int from, to;
        range(rt, from, to);
        if (from >= to) continue;                           // (not staged either)
        if (!mbar_wait(q_full, staged++ & 1, abort_flag)) { fail(ST_TIMEOUT_FULL); break; }
        for (int tile = from; tile < to; ++tile, ++it) {
          const int st = it % ST, b = it & 1;
          ok = (it < 2 || mbar_wait(&s_empty[b], ((it >> 1) - 1) & 1, abort_flag)) && mbar_wait(&k_full[st], (it / ST) & 1, abort_flag);
          if (!ok) { fail(ST_TIMEOUT_FULL); break; }
          tc_fence_after();
          const uint64_t da = dk + uint32_t(st) * (C::K_BYTES / 16);
#pragma unroll
          for (int h = 0; h < KH; ++h) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_f8(tmem + b * NS, da + (h * 1024 + k * 2), dq + (h * (NS * 8) + k * 2), idesc, (h | k) ? 1u : 0u);
          }
          umma_commit(&s_full[b]);
          umma_commit(&k_empty[st]);
        }
      }
    }
  } else {
    const int w = warp >> 2, wq = warp & 3, tl = wq * 32 + lane;
    const uint32_t my_S = tmem + w * NS + (uint32_t(wq * 32) << 16);
    float* out = p.w + seq * p.w_seq + kvh * p.w_head;
    // A wait that runs out does not leave the loop: the warp keeps taking part in the named barriers, without waiting again.
    bool ok = true, staged = false;
    int it = 0;
    for (int rt = 0; rt < n_rt; ++rt) {
      int from, to;
      range(rt, from, to);
      if (from >= to) continue;
      // queries of the tile: one power of two for its rows, two e4m3 terms (as in the decode kernel)
      const int n = min(RN, rows - rt * RN);
      constexpr int CHUNKS = RN * KH * 8, PER = (CHUNKS + 255) / 256;
      const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(p.a.q);
      auto load16 = [&](int i, uint32_t (&u)[8]) {
        const int r = i / (KH * 8), ch = i % (KH * 8);
#pragma unroll
        for (int k = 0; k < 8; ++k) u[k] = 0u;
        if (i < CHUNKS && r < n && ch * 16 < c.dk) {
          const int gr = rt * RN + r;
          const __nv_bfloat16* src = q + long(q0 + first + gr / G) * p.a.q_tok + (kvh * G + gr % G) * p.a.q_head + ch * 16;
          if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
            *reinterpret_cast<uint4*>(u) = reinterpret_cast<const uint4*>(src)[0];
            *reinterpret_cast<uint4*>(u + 4) = reinterpret_cast<const uint4*>(src)[1];
          } else {
            const uint16_t* hs = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
            for (int k = 0; k < 8; ++k) u[k] = hs[2 * k] | uint32_t(hs[2 * k + 1]) << 16;
          }
        }
      };
      uint32_t m = 0;
#pragma unroll 1
      for (int j = 0; j < PER; ++j) {
        uint32_t u[8];
        load16(threadIdx.x + j * 256, u);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t lo = u[k] & 0x7fffu, hi = (u[k] >> 16) & 0x7fffu;
          m = max(m, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
        }
      }
      m = __reduce_max_sync(0xffffffffu, m);
      if (staged) named_sync<3, 256>();            // everybody is through with the rows before, their scores among it
      staged = true;
      if (lane == 0) s_max[warp] = m;
      if (threadIdx.x < RN) {
        const int r = threadIdx.x, gr = rt * RN + r;
        float lse = INFINITY;                      // rows that see nothing or do not exist weigh nothing
        if (r < n) {
          lse = p.a.lse[long(q0 + first + gr / G) * p.a.Hq + kvh * G + gr % G];
          if (lse == -INFINITY) lse = INFINITY;
        }
        s_lse[r] = lse;
        s_pos[r] = r < n ? base + gr / G : -1;
      }
      named_sync<3, 256>();
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, s_max[i]);
      const float qs = kv8_scale_of(__uint_as_float(m << 16)), inv = kv8_inverse(qs);
      const float fq = qs * (CAP ? p.cap_k : p.scale_log2);
#pragma unroll 1
      for (int j = 0; j < PER; ++j) {
        const int i = threadIdx.x + j * 256;
        uint32_t u[8], hi4[4], lo4[4];
        load16(i, u);
        if (i < CHUNKS) {
          const int r = i / (KH * 8), ch = i % (KH * 8);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            hi4[k] = lo4[k] = 0u;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t x = u[2 * k + e];
              const float a0 = __uint_as_float(x << 16) * inv, a1 = __uint_as_float(x & 0xffff0000u) * inv;
              uint32_t hh = e4m3x2(a0, a1);
              if ((x & 0x7f80u) == 0x7f80u) hh |= 0x7fu;
              if ((x & 0x7f800000u) == 0x7f800000u) hh |= 0x7f00u;
              const float2 f = __half22float2(e4m3x2_to_half2(hh));
              hi4[k] |= hh << (16 * e);
              lo4[k] |= e4m3x2((a0 - f.x) * 16.f, (a1 - f.y) * 16.f) << (16 * e);
            }
          }
          uint8_t* dst = q_s + (ch / 8) * (NS * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
          *reinterpret_cast<uint4*>(dst) = make_uint4(hi4[0], hi4[1], hi4[2], hi4[3]);
          *reinterpret_cast<uint4*>(dst + RN * 128) = make_uint4(lo4[0], lo4[1], lo4[2], lo4[3]);
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(q_full);

      const int pos_a = base + rt * RN / G, pos_b = base + (min(rows, (rt + 1) * RN) - 1) / G;
      for (int tile = from; tile < to; ++tile, ++it) {
        if ((it & 1) != w) continue;
        const int tok = tile * BKV + tl;
        float ks = 0.f, old = 0.f;
        if (tok < ctx) {
          const int blk = bt[tok / c.page];
          if (unsigned(blk) < unsigned(c.n_blocks)) ks = c.k_scale[long(blk) * c.Hkv + kvh];
          else atomicCAS(p.s.status, 0, ST_BAD_ARGS);
          old = out[tok];
        }
        const float mul = fq * ks;
        if (ok && !__all_sync(0xffffffffu, mbar_wait(&s_full[w], (it >> 1) & 1, abort_flag))) ok = fail(ST_TIMEOUT_TMEM_FULL);
        if (!ok) continue;
        tc_fence_after();
        const bool full = tile * BKV + BKV <= min(ctx, pos_a + 1) && (p.a.window == 0 || tile * BKV > pos_b - p.a.window);
        float acc0 = 0.f, acc1 = 0.f;
#pragma unroll
        for (int r0 = 0; r0 < RN; r0 += 8) {
          uint32_t h8[8], l8[8];
          asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                       : "=r"(h8[0]), "=r"(h8[1]), "=r"(h8[2]), "=r"(h8[3]), "=r"(h8[4]), "=r"(h8[5]), "=r"(h8[6]), "=r"(h8[7])
                       : "r"(my_S + r0) : "memory");
          asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                       : "=r"(l8[0]), "=r"(l8[1]), "=r"(l8[2]), "=r"(l8[3]), "=r"(l8[4]), "=r"(l8[5]), "=r"(l8[6]), "=r"(l8[7])
                       : "r"(my_S + RN + r0) : "memory");
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float s = fmaf(__uint_as_float(l8[j]), 0.0625f, __uint_as_float(h8[j])) * mul;
            if constexpr (CAP) s = fmaf(softcap_r(s, 1.f), p.scale_log2, 0.5f * p.scale_log2);
            float y = ex2(s - s_lse[r0 + j]);
            if (!full) {
              const int pos = s_pos[r0 + j];
              if (tok > pos || (p.a.window > 0 && tok <= pos - p.a.window)) y = 0.f;
            }
            if (j & 1) acc1 += y;
            else acc0 += y;
          }
        }
        tc_fence_before();
        mbar_arrive(&s_empty[w]);
        if (tok < ctx) out[tok] = old + (acc0 + acc1);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

template <int KH, int RN, bool CAP>
cudaError_t launch(const CUtensorMap* tk, const WeightArgs& p, int n_splits, cudaStream_t st) {
  auto kfn = kv8_weights_kernel<KH, RN, CAP>;
  static DeviceOnce once;
  const cudaError_t e = once.shared_memory(reinterpret_cast<const void*>(kfn), WCfg<KH, RN>::SMEM);
  if (e != cudaSuccess) return e;
  return launch_pdl(kfn, dim3(p.c.Hkv, n_splits, p.s.n), dim3(320), WCfg<KH, RN>::SMEM, st, *tk, p);
}

}  // namespace

int kv8_weights_launch(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Attn& a, int observe, int per, int n_splits, float* w, long w_seq,
                       long w_head, int w_keys, cudaStream_t st) {
  if (s.n <= 0 || s.T <= 0 || s.max_new <= 0) return 0;
  const CUtensorMap* tk = tmap_2d(c.k, uint64_t(c.n_blocks) * c.Hkv * c.page, c.dk, c.dk, c.page, 128, TM_U8, true);
  if (!tk) {
    kv8_set_error(tmap_last_error());
    return 1;
  }
  WeightArgs p{c, s, a, observe, per, a.scale * 1.4426950408889634f, 0.f, w, w_seq, w_head, w_keys};
  const bool cap = a.softcap > 0.f;
  if (cap) {
    p.cap_k = 2.f * 1.4426950408889634f * a.scale / a.softcap;
    p.scale_log2 = 2.f * 1.4426950408889634f * a.softcap;
  }
  const long rows = long(observe > 0 && observe < s.max_new ? observe : s.max_new) * (a.Hq / c.Hkv);
  const int kh = (c.dk + 127) / 128, rn = rows <= 8 ? 8 : (rows <= 16 ? 16 : 64);
  cudaError_t e = cudaErrorInvalidValue;
#define LB_KV8(K_, R_) \
  if (kh == K_ && rn == R_) e = cap ? launch<K_, R_, true>(tk, p, n_splits, st) : launch<K_, R_, false>(tk, p, n_splits, st);
  LB_KV8(1, 8) LB_KV8(1, 16) LB_KV8(1, 64) LB_KV8(2, 8) LB_KV8(2, 16) LB_KV8(2, 64)
#undef LB_KV8
  if (e != cudaSuccess) kv8_set_error(cudaGetErrorString(e));
  return e != cudaSuccess;
}

}  // namespace lb
