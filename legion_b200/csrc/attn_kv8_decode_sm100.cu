// Decode attention over the 8-bit key/value cache on tcgen05 for sm_100a: one query row per sequence, the query heads of a kv
// head share every byte.
//
// The codes go from TMA into kind::f8f6f4 MMAs as they are, keys as the UMMA M dimension (tiles of 128):
//     S^T[128 keys, heads] = K[128, D] . Q^T          (K tile: K-major A operand)
//     O^T[D, heads]       += V^T[D, 128 keys] . P     (V tile: MN-major A operand, same TMA layout)
// and the other operand is split into 8-bit terms that lie side by side in the N dimension, which a decode step has to spare:
//   * a query times a power of two is  hi + lo / 16  in e4m3, exactly: 8 bits of a bf16 value = 4 + 4;
//   * a probability is  t1 + t2 + t3  in e5m2, 9 bits over the range of a half. e5m2 is the upper byte of a half, so a term
//     turns back into a half by a byte move and the remainder is one exact half subtraction.
// Scales never touch the codes: a key's scale multiplies its score, and a value's scale 2^e joins the exponent, z = s + e, so
// that the running reference is the largest weight a code can get, P stays in the range of a half whatever the scales are, and
// the denominator adds exp(z) 2^-e.
//
// Two softmax warpgroups (warps 0..3 and 4..7; thread = key of the tile, later output column) take alternate tiles, each a
// stream of its own with its P and O^T; they meet in shared memory at the end. Warp 8: MMAs, scores four tiles ahead of
// their softmax (a wait for a phase of a stage's barrier cannot miss it: the stage's next scores stand behind P of this tile, the
// stage's next P V behind P of the tile that waits). Warp 9: TMA through the block table into as many stages as 192 KB hold (six of 32 KB for heads of 128), which
// is what a memory-bound kernel needs in flight. Splits of a sequence write partial results for kv8_combine_kernel; a split
// covers the same number of tiles in every sequence, so CTAs of a ragged batch are alike. Scratch belongs to the call.
#include "kv8_dev.cuh"
#include "tmap.cuh"

namespace lb {
namespace {

struct DecodeArgs {
  Kv8Cache c;
  Kv8Seqs s;
  Kv8Attn a;
  int per, n_splits;
  float scale_log2, cap_k;      // as in softcap_r: soft-capped scores have 2 cap log2(e) in scale_log2
  float* part;                  // [T][Hq][n_splits][dv + 2]: sums over the values, reference (log2), denominator
};

// P is taken relative to the reference times 2^11, and the reference moves when a weight passes it by more than 2^4: at most 2^15,
// which e5m2 and a half hold, and e5m2's last step, 2^-16, lies 2^-27 below the largest weight. (A reference within 2^2 moved in a
// quarter of the tiles of a stream of 2000 keys, 1900 clocks each.)
constexpr float OFFSET = 11.f;
constexpr float SLACK = 4.f;

__device__ __forceinline__ int ordered(float f) {
  const int i = __float_as_int(f);
  return i >= 0 ? i : i ^ 0x7fffffff;
}
__device__ __forceinline__ float unordered(int i) { return __int_as_float(i >= 0 ? i : i ^ 0x7fffffff); }

template <int N>
__device__ __forceinline__ void tm_ld(uint32_t at, uint32_t* r) {
  static_assert(N % 16 == 0, "columns");
#pragma unroll
  for (int i = 0; i < N; i += 16) tmem_ld16(at + i, *reinterpret_cast<uint32_t(*)[16]>(r + i));
}
__device__ __forceinline__ void tm_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
template <int BAR, int N>
__device__ __forceinline__ void named_sync() {
  asm volatile("bar.sync %0, %1;" ::"n"(BAR), "n"(N) : "memory");
}

// KH, MT: 128-column parts of a key and of a value; NQ: query heads of a CTA
template <int KH, int MT, int NQ>
struct Cfg {
  static constexpr int BKV = 128;
  static constexpr int NS = 2 * NQ, NO = (3 * NQ + 15) / 16 * 16;
  static constexpr int K_BYTES = KH * BKV * 128, V_BYTES = MT * BKV * 128;
  static constexpr int STAGES = 192 * 1024 / (K_BYTES + V_BYTES);          // 6, 4 or 3
  static constexpr int Q_BYTES = KH * NS * 128, P_BYTES = NO * 128;
  static constexpr int O_BYTES = NQ * MT * 128 * 4;                        // the second warpgroup's sums on their way to the first
  static constexpr int TAIL = 1024;
  static constexpr int SMEM = STAGES * (K_BYTES + V_BYTES) + Q_BYTES + 2 * P_BYTES + TAIL + 1024;
  static constexpr int LA = STAGES < 4 ? STAGES : 4;                       // tiles whose scores are made ahead
  static constexpr int TMEM_RAW = LA * NS + 2 * MT * NO;
  static constexpr int TMEM_COLS = TMEM_RAW <= 128 ? 128 : TMEM_RAW <= 256 ? 256 : 512;
  static_assert(TMEM_RAW <= 512 && STAGES >= 3 && STAGES <= 6 && SMEM <= 227 * 1024 && O_BYTES <= K_BYTES, "sizes");
};

template <int KH, int MT, int NQ, bool CAP>
__global__ void __launch_bounds__(320, 1)
kv8_decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const DecodeArgs p) {
  using C = Cfg<KH, MT, NQ>;
  constexpr int BKV = C::BKV, NS = C::NS, NO = C::NO, ST = C::STAGES, LA = C::LA;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* k_s = smem;
  uint8_t* v_s = k_s + ST * C::K_BYTES;
  uint8_t* q_s = v_s + ST * C::V_BYTES;
  uint8_t* p_s = q_s + C::Q_BYTES;                        // [2], each on 1024 bytes
  uint64_t* bars = reinterpret_cast<uint64_t*>(p_s + 2 * C::P_BYTES);
  uint64_t* k_full = bars;         // [6] one per stage
  uint64_t* k_done = bars + 6;     // scores made: for the softmax, and the stage is free
  uint64_t* v_full = bars + 12;
  uint64_t* v_done = bars + 18;    // P V done: P may be written, O touched, and the stage is free
  uint64_t* p_ready = bars + 24;   // [2] one per warpgroup
  uint64_t* q_full = bars + 30;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 31);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* s_red = reinterpret_cast<float*>(bars + 32);     // [2 warpgroups][NQ][4 warps] maxima, then sums

  const Kv8Cache& c = p.c;
  const int G = p.a.Hq / c.Hkv, gtiles = (G + NQ - 1) / NQ;
  const int kvh = blockIdx.x / gtiles, g0 = (blockIdx.x % gtiles) * NQ, gn = min(NQ, G - g0), head0 = kvh * G + g0;
  const int b = blockIdx.y, split = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  griddep_wait();
  griddep_launch();
  const int row = p.s.cu[b];
  if (p.s.cu[b + 1] <= row) return;
  if (row < 0 || row >= p.s.T || p.s.cu[b + 1] != row + 1) {
    if (threadIdx.x == 0) atomicCAS(p.s.status, 0, ST_BAD_ARGS);
    return;
  }
  const int ctx = int(min(long(max(p.s.ctx[b], 0)), long(p.s.width) * c.page));
  const int start = (p.a.window > 0 && ctx > p.a.window) ? ctx - p.a.window : 0;
  const int tile0 = start / BKV + split * p.per, tiles_end = (ctx + BKV - 1) / BKV;
  const int tile1 = split == p.n_splits - 1 ? tiles_end : min(tiles_end, tile0 + p.per);   // (longer than announced: the last takes the rest)
  const int n_tiles = tile1 - tile0;
  const int D = c.dv;
  float* part = p.n_splits > 1 ? p.part + ((long(row) * p.a.Hq + head0) * p.n_splits + split) * (D + 2) : nullptr;
  const long part_head = long(p.n_splits) * (D + 2);
  if (n_tiles <= 0) {
    if (split > 0 || part) return;                        // the merge counts the splits that have tiles
    for (int i = threadIdx.x; i < gn * D; i += blockDim.x)
      static_cast<__nv_bfloat16*>(p.a.out)[row * p.a.o_tok + (head0 + i / D) * D + i % D] = __float2bfloat16(0.f);
    if (p.a.lse && threadIdx.x < gn) p.a.lse[long(row) * p.a.Hq + head0 + threadIdx.x] = -INFINITY;
    return;
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_done[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_done[i], 1);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&p_ready[i], 128);
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
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t tmem_S = tmem_base, tmem_O = tmem_base + LA * NS;
  const int* bt = p.s.table + b * p.s.ld_table;
  const int ppb = BKV / c.page;

  if (warp == 9) {
    // ------------------------------------------------------------------ TMA: the lanes fetch the table, lane 0 issues
    const int tiles_per_fill = 32 / ppb;
    int pg_reg = 0;
    bool ok = true;
    for (int i = 0; ok && i < n_tiles; ++i) {
      const int slot = i % tiles_per_fill;
      if (slot == 0) {
        const long page = long(tile0 + i) * ppb + lane;
        // pages behind the sequence: a block outside the cache, whose rows TMA fills with zeros
        pg_reg = page * c.page < ctx ? bt[page] : c.n_blocks;
        if (unsigned(pg_reg) > unsigned(c.n_blocks)) pg_reg = c.n_blocks;
      }
      const int st = i % ST;
      for (int kv = 0; ok && kv < 2; ++kv) {
        uint64_t* empty = kv ? &v_done[st] : &k_done[st];
        uint64_t* full = kv ? &v_full[st] : &k_full[st];
        if (i >= ST && !__all_sync(0xffffffffu, mbar_wait(empty, ((i / ST) - 1) & 1, abort_flag))) {
          if (lane == 0) { *abort_flag = 1; atomicCAS(p.s.status, 0, ST_TIMEOUT_EMPTY | SITE_DECODE_ATTN); }
          ok = false;
          break;
        }
        uint8_t* dst = kv ? v_s + st * C::V_BYTES : k_s + st * C::K_BYTES;
        if (lane == 0) mbar_expect_tx(full, kv ? C::V_BYTES : C::K_BYTES);
        for (int g = 0; g < ppb; ++g) {
          const int pg = __shfl_sync(0xffffffffu, pg_reg, slot * ppb + g);
          if (lane == 0) {
            for (int h = 0; h < (kv ? MT : KH); ++h)
              tma_load_2d(dst + h * (BKV * 128) + g * c.page * 128, kv ? &tmV : &tmK, full, h * 128, (pg * c.Hkv + kvh) * c.page);
          }
        }
      }
    }
  } else if (warp == 8) {
    // ------------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      constexpr uint32_t idesc_s = umma_idesc(128, NS, 0, 0, 0, 0);       // e4m3 x e4m3
      constexpr uint32_t idesc_o = umma_idesc(128, NO, 0, 1, 1, 0);       // e4m3 (V^T, MN-major) x e5m2
      // Descriptors are made once; a step adds its offset in 16-byte units. (Made anew for every MMA they take the one issuing
      // thread 170 clocks each; an MMA of this shape takes 40.)
      const uint64_t dk = umma_desc_k_sw128(smem_u32(k_s)), dq = umma_desc_k_sw128(smem_u32(q_s));
      const uint64_t dv = umma_desc_mn_sw128(smem_u32(v_s), BKV * 128, 1024), dp = umma_desc_k_sw128(smem_u32(p_s));
      auto fail = [&](int code) { *abort_flag = 1; atomicCAS(p.s.status, 0, code | SITE_DECODE_ATTN); return false; };
      auto issue_s = [&](int i) -> bool {
        const int st = i % ST;
        if (!mbar_wait(&k_full[st], (i / ST) & 1, abort_flag)) return fail(ST_TIMEOUT_FULL);
        tc_fence_after();
        const uint64_t da = dk + uint32_t(st) * (C::K_BYTES / 16);
        const uint32_t ts = tmem_S + (i % LA) * NS;
#pragma unroll
        for (int h = 0; h < KH; ++h) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f8(ts, da + (h * (BKV * 8) + k * 2), dq + (h * (NS * 8) + k * 2), idesc_s, (h | k) ? 1u : 0u);
        }
        umma_commit(&k_done[st]);
        return true;
      };
      bool ok = mbar_wait(q_full, 0, abort_flag) || fail(ST_TIMEOUT_FULL);
      for (int i = 0; ok && i < min(LA, n_tiles); ++i) ok = issue_s(i);
      for (int i = 0; ok && i < n_tiles; ++i) {
        const int w = i & 1, st = i % ST;
        if (!mbar_wait(&p_ready[w], (i >> 1) & 1, abort_flag)) { fail(ST_TIMEOUT_FLAG); break; }
        if (!mbar_wait(&v_full[st], (i / ST) & 1, abort_flag)) { fail(ST_TIMEOUT_FULL); break; }
        tc_fence_after();
        const uint64_t da = dv + uint32_t(st) * (C::V_BYTES / 16), db = dp + uint32_t(w) * (C::P_BYTES / 16);
        const uint32_t to = tmem_O + w * MT * NO;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int k = 0; k < BKV / 32; ++k)
            umma_f8(to + mt * NO, da + (mt * (BKV * 8) + k * 256), db + k * 2, idesc_o, ((i >> 1) | k) ? 1u : 0u);
        }
        umma_commit(&v_done[st]);
        if (i + LA < n_tiles && !issue_s(i + LA)) break;      // into the buffer of tile i, which its softmax has read
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax (warps 0..7)
    const int w = warp >> 2, wq = warp & 3, tl = wq * 32 + lane;
    const uint32_t lane_off = uint32_t(wq * 32) << 16;
    const uint32_t my_S = tmem_S + lane_off, my_O = tmem_O + w * MT * NO + lane_off;
    const int bar_id = 1 + w;
    float* red = s_red + w * (NQ * 4);
    uint8_t* my_p = p_s + w * C::P_BYTES;

    // queries: one power of two for all heads of the CTA (what a smaller head loses is 2^-21 of the largest query value, and a
    // softmax sees absolute errors of its scores); a value that is not finite is a NaN code and makes its head NaN
    float fq;
    {
      constexpr int CHUNKS = NQ * KH * 8;                  // of 16 values
      const int q = threadIdx.x / (KH * 8), ch = threadIdx.x % (KH * 8);
      uint32_t u[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] = 0u;
      uint32_t m = 0;
      if (threadIdx.x < CHUNKS && q < gn && ch * 16 < c.dk) {
        const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(p.a.q) + row * p.a.q_tok + (head0 + q) * p.a.q_head + ch * 16;
        if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
          *reinterpret_cast<uint4*>(u) = reinterpret_cast<const uint4*>(src)[0];
          *reinterpret_cast<uint4*>(u + 4) = reinterpret_cast<const uint4*>(src)[1];
        } else {
          const uint16_t* hsrc = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
          for (int i = 0; i < 8; ++i) u[i] = hsrc[2 * i] | uint32_t(hsrc[2 * i + 1]) << 16;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t lo = u[i] & 0x7fffu, hi = (u[i] >> 16) & 0x7fffu;
          m = max(m, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
        }
      }
      m = __reduce_max_sync(0xffffffffu, m);
      uint32_t* s_m = reinterpret_cast<uint32_t*>(s_red);
      if (lane == 0) s_m[warp] = m;
      named_sync<3, 256>();
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, s_m[i]);
      named_sync<3, 256>();
      const float qs = kv8_scale_of(__uint_as_float(m << 16));
      const float inv = kv8_inverse(qs);
      fq = qs * p.scale_log2;
      if (CAP) fq = qs * p.cap_k;
      if (threadIdx.x < CHUNKS) {
        uint32_t hi4[4], lo4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          hi4[i] = lo4[i] = 0u;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t x = u[2 * i + j];
            const float a0 = __uint_as_float(x << 16) * inv, a1 = __uint_as_float(x & 0xffff0000u) * inv;
            uint32_t hh = e4m3x2(a0, a1);
            if ((x & 0x7f80u) == 0x7f80u) hh |= 0x7fu;
            if ((x & 0x7f800000u) == 0x7f800000u) hh |= 0x7f00u;
            const float2 f = __half22float2(e4m3x2_to_half2(hh));
            hi4[i] |= hh << (16 * j);
            lo4[i] |= e4m3x2((a0 - f.x) * 16.f, (a1 - f.y) * 16.f) << (16 * j);
          }
        }
        const uint32_t at = (ch / 8) * (NS * 128) + q * 128 + (((ch & 7) ^ (q & 7)) << 4);
        *reinterpret_cast<uint4*>(q_s + at) = make_uint4(hi4[0], hi4[1], hi4[2], hi4[3]);
        *reinterpret_cast<uint4*>(q_s + at + NQ * 128) = make_uint4(lo4[0], lo4[1], lo4[2], lo4[3]);
      }
    }
    for (int j = tl; j < C::P_BYTES / 16; j += 128) reinterpret_cast<uint4*>(my_p)[j] = make_uint4(0u, 0u, 0u, 0u);
    fence_proxy_async_smem();
    mbar_arrive(q_full);

    float m_ref[NQ], l_run[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) { m_ref[q] = -INFINITY; l_run[q] = 0.f; }
    // this thread's key of a tile: scales of its block
    auto scales = [&](int tile, float& ks, float& vs) {
      const int tok = tile * BKV + tl;
      ks = vs = 0.f;
      if (tok < ctx) {
        const int blk = bt[tok / c.page];
        if (unsigned(blk) < unsigned(c.n_blocks)) {
          const long u = long(blk) * c.Hkv + kvh;
          ks = c.k_scale[u];
          vs = c.v_scale[u];
        } else {
          atomicCAS(p.s.status, 0, ST_BAD_ARGS);
        }
      }
    };
    bool ok = true;
    auto fail = [&](int code) { *abort_flag = 1; atomicCAS(p.s.status, 0, code | SITE_DECODE_ATTN); ok = false; };
    float ks = 0.f, vs = 0.f;
    if (w < n_tiles) scales(tile0 + w, ks, vs);
    int n_mine = 0;
    for (int i = w; i < n_tiles; i += 2, ++n_mine) {
      const float mul = fq * ks;
      const int ev = kv8_log2(vs);
      const float add = float(ev), inv_v = __uint_as_float(uint32_t(127 - ev) << 23);     // |ev| <= 120
      if (i + 2 < n_tiles) scales(tile0 + i + 2, ks, vs);       // the next tile's, while this one is worked on
      if (ok && !__all_sync(0xffffffffu, mbar_wait(&k_done[i % ST], (i / ST) & 1, abort_flag))) fail(ST_TIMEOUT_TMEM_FULL);
      uint32_t r[NS];
#pragma unroll
      for (int q = 0; q < NS; ++q) r[q] = 0u;
      if (ok) {
        tc_fence_after();
        tm_ld<NS>(my_S + (i % LA) * NS, r);
        tmem_ld_wait();
      }
      const int key0 = (tile0 + i) * BKV, tok = key0 + tl;
      const bool valid = tok >= start && tok < ctx;
      float z[NQ];
      bool over = false;
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        z[q] = -INFINITY;
        if (q < gn) {
          float s = fmaf(__uint_as_float(r[NQ + q]), 0.0625f, __uint_as_float(r[q])) * mul;
          if constexpr (CAP) s = fmaf(softcap_r(s, 1.f), p.scale_log2, 0.5f * p.scale_log2);
          if (valid) z[q] = s + add;
          over |= z[q] > m_ref[q] + SLACK;
        }
      }
      uint32_t any_over;
      asm volatile(
          "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, %2, 128, p;\n\t"
          "selp.u32 %0, 1, 0, q;\n\t}"
          : "=r"(any_over) : "r"(over ? 1u : 0u), "r"(bar_id) : "memory");
      if (ok && n_mine >= 1 && !__all_sync(0xffffffffu, mbar_wait(&v_done[(i - 2) % ST], ((i - 2) / ST) & 1, abort_flag)))
        fail(ST_TIMEOUT_TMEM_EMPTY);
      if (any_over) {
        float alpha[NQ];
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          if (q < gn) {
            const int wm = __reduce_max_sync(0xffffffffu, ordered(z[q]));
            if (lane == q) red[q * 4 + wq] = unordered(wm);
          }
        }
        asm volatile("bar.sync %0, 128;" ::"r"(bar_id) : "memory");
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          alpha[q] = 1.f;
          if (q < gn) {
            const float4 m4 = *reinterpret_cast<const float4*>(&red[q * 4]);
            const float m = fmaxf(fmaxf(m4.x, m4.y), fmaxf(m4.z, m4.w));
            if (m > m_ref[q]) {
              alpha[q] = m_ref[q] == -INFINITY ? 0.f : ex2(m_ref[q] - m);
              m_ref[q] = m;
            }
            l_run[q] *= alpha[q];
          }
        }
        if (ok && n_mine >= 1) {
          tc_fence_after();
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            uint32_t o[NO];
            tm_ld<NO>(my_O + mt * NO, o);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 3 * NQ; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha[j % NQ]);
#pragma unroll
            for (int j = 0; j < NO; j += 16) tm_st16(my_O + mt * NO + j, o + j);
          }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        }
        asm volatile("bar.sync %0, 128;" ::"r"(bar_id) : "memory");      // red is read before it is written again
      }
      // P: [term * NQ + head][key], K-major rows of 128 bytes, 128-byte swizzle
#pragma unroll
      for (int q = 0; q < NQ; q += 2) {
        if (q < gn) {
          float y[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float ref = m_ref[q + e] == -INFINITY ? 0.f : m_ref[q + e] - OFFSET;
            y[e] = ex2(z[q + e] - ref);
            l_run[q + e] = fmaf(y[e], inv_v, l_run[q + e]);
          }
          __half2 h = __floats2half2_rn(y[0], y[1]);
#pragma unroll
          for (int t = 0; t < 3; ++t) {
            const uint32_t b2 = e5m2x2(h);
            if (t < 2) h = __hsub2(h, e5m2x2_to_half2(b2));
            const int c16 = tl >> 4;
            my_p[(t * NQ + q) * 128 + ((c16 ^ (q & 7)) << 4) + (tl & 15)] = uint8_t(b2);
            my_p[(t * NQ + q + 1) * 128 + ((c16 ^ ((q + 1) & 7)) << 4) + (tl & 15)] = uint8_t(b2 >> 8);
          }
        }
      }
      // values of keys that nobody sees (in front of the window, behind the sequence) may hold anything, a NaN code too, which
      // a zero probability would not cancel
      if (key0 < start || key0 + BKV > ctx) {
        const int st = i % ST;
        if (ok && !__all_sync(0xffffffffu, mbar_wait(&v_full[st], (i / ST) & 1, abort_flag))) fail(ST_TIMEOUT_FULL);
        if (ok && !valid) {
#pragma unroll
          for (int j = 0; j < MT * 8; ++j)
            *reinterpret_cast<uint4*>(v_s + st * C::V_BYTES + (j / 8) * (BKV * 128) + tl * 128 + (j % 8) * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
      }
      fence_proxy_async_smem();
      tc_fence_before();
      mbar_arrive(&p_ready[w]);
    }
    if (ok && n_mine >= 1) {
      const int last = w + 2 * (n_mine - 1);
      if (!__all_sync(0xffffffffu, mbar_wait(&v_done[last % ST], (last / ST) & 1, abort_flag))) fail(ST_TIMEOUT_TMEM_FULL);
    }
    // sums over the keys; the second warpgroup hands its results to the first through the (now idle) key stages
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      float v = l_run[q];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (lane == q) red[q * 4 + wq] = v;
    }
    named_sync<3, 256>();
    float l[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const float4 s4 = *reinterpret_cast<const float4*>(&red[q * 4]);
      l[q] = (s4.x + s4.y) + (s4.z + s4.w);
    }
    float* o_x = reinterpret_cast<float*>(k_s);           // [MT * 128][NQ]
    float* ml_x = reinterpret_cast<float*>(q_s);          // [NQ][2]
    float acc[MT][NQ];
    tc_fence_after();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      uint32_t o[NO];
#pragma unroll
      for (int j = 0; j < NO; ++j) o[j] = 0u;
      if (ok && n_mine >= 1) {
        tm_ld<NO>(my_O + mt * NO, o);
        tmem_ld_wait();
      }
#pragma unroll
      for (int q = 0; q < NQ; ++q)
        acc[mt][q] = __uint_as_float(o[q]) + (__uint_as_float(o[NQ + q]) + __uint_as_float(o[2 * NQ + q]));
    }
    if (w == 1) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int q = 0; q < NQ; ++q) o_x[(q * MT + mt) * 128 + tl] = acc[mt][q];
      }
      if (tl == 0) {
#pragma unroll
        for (int q = 0; q < NQ; ++q) { ml_x[2 * q] = m_ref[q]; ml_x[2 * q + 1] = l[q]; }
      }
    }
    named_sync<3, 256>();
    if (w == 0 && !*abort_flag) {
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        if (q < gn) {
          const float m1 = ml_x[2 * q], l1 = ml_x[2 * q + 1];
          const float m = fmaxf(m_ref[q], m1);
          const float f0 = m_ref[q] == -INFINITY ? (l[q] == l[q] ? 0.f : 1.f) : ex2(m_ref[q] - m);      // (NaN passes)
          const float f1 = m1 == -INFINITY ? (l1 == l1 ? 0.f : 1.f) : ex2(m1 - m);
          const float ll = l[q] * f0 + l1 * f1;
          const float ref = m == -INFINITY ? m : m - OFFSET;
          float inv = 0.f;
          if (!part) {
            float den = ll, top = ref;
            if (p.a.sink) {
              const float sk = p.a.sink[head0 + q] * 1.4426950408889634f;
              if (top == -INFINITY) { top = sk; den = 1.f; }
              else den += ex2(sk - top);
            }
            inv = den > 0.f || den != den ? 1.f / den : 0.f;
            if (p.a.lse && tl == 0) p.a.lse[long(row) * p.a.Hq + head0 + q] = den > 0.f ? top + log2f(den) : -INFINITY;
          } else if (tl == 0) {
            part[q * part_head + D] = ref;
            part[q * part_head + D + 1] = ll;
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            const int d = mt * 128 + tl;
            const float o = acc[mt][q] * f0 + o_x[(q * MT + mt) * 128 + tl] * f1;
            if (d < D) {
              if (part) part[q * part_head + d] = o;
              else static_cast<__nv_bfloat16*>(p.a.out)[row * p.a.o_tok + (head0 + q) * D + d] = __float2bfloat16(o * inv);
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
}

// Joins the splits of a row and head: sum over splits of 2^(m - M) O, over the sum of 2^(m - M) l (and a sink). Splits of a decode
// row that got no tiles left no partial results; those of prompt rows (ROWS: one CTA per row and head) all did.
template <bool ROWS>
__global__ void __launch_bounds__(128) kv8_combine_kernel(const DecodeArgs p) {
  __shared__ float s_w[129];
  griddep_wait();
  griddep_launch();
  const int D = p.c.dv, h = blockIdx.x % p.a.Hq;
  long row = blockIdx.x / p.a.Hq;
  int live = p.n_splits;
  if (!ROWS) {
    const int b = int(row);
    row = p.s.cu[b];
    if (p.s.cu[b + 1] != row + 1 || row < 0 || row >= p.s.T) return;
    const int ctx = int(min(long(max(p.s.ctx[b], 0)), long(p.s.width) * p.c.page));
    const int start = (p.a.window > 0 && ctx > p.a.window) ? ctx - p.a.window : 0;
    live = min(p.n_splits, ((ctx + 127) / 128 - start / 128 + p.per - 1) / p.per);
  } else if (row < p.s.cu[0] || row >= p.s.cu[p.s.n]) {
    return;                                                 // a row of no sequence
  }
  const float* part = p.part + (long(row) * p.a.Hq + h) * p.n_splits * (D + 2);
  const float sk = p.a.sink ? p.a.sink[h] * 1.4426950408889634f : -INFINITY;
  if (threadIdx.x < 32) {
    float m = sk;
    for (int i = threadIdx.x; i < live; i += 32) m = fmaxf(m, part[long(i) * (D + 2) + D]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float l = 0.f;
    for (int i = threadIdx.x; i < live; i += 32) {
      const float mi = part[long(i) * (D + 2) + D], li = part[long(i) * (D + 2) + D + 1];
      const float f = mi == -INFINITY ? (li == li ? 0.f : 1.f) : ex2(mi - m);
      l += f * li;
      s_w[i] = f;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (sk != -INFINITY) l += ex2(sk - m);
    if (threadIdx.x == 0) {
      s_w[128] = l > 0.f || l != l ? 1.f / l : 0.f;
      if (p.a.lse) p.a.lse[long(row) * p.a.Hq + h] = l > 0.f ? m + log2f(l) : -INFINITY;
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += 128) {
    float o = 0.f;
#pragma unroll 4
    for (int i = 0; i < live; ++i) o += s_w[i] * part[long(i) * (D + 2) + d];
    static_cast<__nv_bfloat16*>(p.a.out)[row * p.a.o_tok + h * D + d] = __float2bfloat16(o * s_w[128]);
  }
}

template <int KH, int MT, int NQ, bool CAP>
cudaError_t launch(const CUtensorMap* tk, const CUtensorMap* tv, const DecodeArgs& p, cudaStream_t st) {
  auto kfn = kv8_decode_kernel<KH, MT, NQ, CAP>;
  constexpr int smem = Cfg<KH, MT, NQ>::SMEM;
  static DeviceOnce once;
  const cudaError_t e = once.shared_memory(reinterpret_cast<const void*>(kfn), smem);
  if (e != cudaSuccess) return e;
  const int G = p.a.Hq / p.c.Hkv;
  return launch_pdl(kfn, dim3(p.c.Hkv * ((G + NQ - 1) / NQ), p.s.n, p.n_splits), dim3(320), smem, st, *tk, *tv, p);
}

}  // namespace

cudaError_t kv8_join(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Attn& a, int n_splits, float* part, cudaStream_t st) {
  const DecodeArgs p{c, s, a, 0, n_splits, 0.f, 0.f, part};
  kv8_combine_kernel<true><<<unsigned(s.T * a.Hq), 128, 0, st>>>(p);
  return cudaGetLastError();
}

int kv8_decode_launch(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Attn& a, int per, int n_splits, float* part, cudaStream_t st) {
  if (s.n <= 0 || s.T <= 0) return 0;
  const uint64_t rows = uint64_t(c.n_blocks) * c.Hkv * c.page;
  const CUtensorMap* tk = tmap_2d(c.k, rows, c.dk, c.dk, c.page, 128, TM_U8, true);
  const CUtensorMap* tv = tmap_2d(c.v, rows, c.dv, c.dv, c.page, 128, TM_U8, true);
  if (!tk || !tv) {
    kv8_set_error(tmap_last_error());
    return 1;
  }
  DecodeArgs p{c, s, a, per, n_splits, a.scale * 1.4426950408889634f, 0.f, part};
  const bool cap = a.softcap > 0.f;
  if (cap) {
    p.cap_k = 2.f * 1.4426950408889634f * a.scale / a.softcap;
    p.scale_log2 = 2.f * 1.4426950408889634f * a.softcap;
  }
  const int kh = (c.dk + 127) / 128, mt = (c.dv + 127) / 128, nq = a.Hq / c.Hkv <= 8 ? 8 : 16;
  cudaError_t e = cudaErrorInvalidValue;
#define LB_KV8(K_, V_, Q_) \
  if (kh == K_ && mt == V_ && nq == Q_) e = cap ? launch<K_, V_, Q_, true>(tk, tv, p, st) : launch<K_, V_, Q_, false>(tk, tv, p, st);
  LB_KV8(1, 1, 8) LB_KV8(1, 1, 16) LB_KV8(2, 2, 8) LB_KV8(2, 2, 16) LB_KV8(1, 2, 8) LB_KV8(1, 2, 16) LB_KV8(2, 1, 8) LB_KV8(2, 1, 16)
#undef LB_KV8
  if (e == cudaSuccess && n_splits > 1) e = launch_pdl(kv8_combine_kernel<false>, dim3(unsigned(a.Hq) * s.n), dim3(128), 0, st, p);
  if (e != cudaSuccess) kv8_set_error(cudaGetErrorString(e));
  return e != cudaSuccess;
}

}  // namespace lb
