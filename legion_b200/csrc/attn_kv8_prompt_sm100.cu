// Prompt attention over the 8-bit key/value cache on tcgen05 for sm_100a.
//
// The query heads of a kv head share its keys, so rows are packed: row r of a sequence and kv head is token r / G, head r % G, and
// one CTA takes RT tiles of 128 such rows (two where values have at most 128 columns) over tiles of 128 keys:
//     S = Q K^T    kind::f8f6f4, the codes as TMA brings them; a query row times a power of two is hi + lo in e4m3 (8 bits of a
//                  bf16 value = 4 + 4, down to 2^-17 of the row's largest), lo as further K steps of the same accumulator: as many
//                  MMA cycles as bf16 operands would take
//     O += P V     kind::f16: P as halves in tensor memory over the scores it came from, V expanded to halves by a warpgroup of
//                  its own. Splitting P into 8-bit terms instead would cost the softmax threads, which bound this kernel, four
//                  instructions per element; V has as many elements per key tile as one row tile's P, and two tiles share it.
// A key's scale multiplies its score, a value's scale 2^e joins the exponent, z = s + e, and the running reference is taken over
// z, so P stays in the range of a half; the denominator adds exp(z) 2^-e. Both come per 8 keys from a ring in shared memory.
//
// 8192 tokens, 32 / 4 heads of 128: 730 us = 753 TFLOP/s, 0.45 of the measured bf16 rate. A pair of row tiles and 128 keys take 4400
// clocks, tensor cores and exponentials 2050 each: a row tile's softmax, P V and next scores follow one another (two score tiles
// and two outputs fill tensor memory), and score MMAs run at shared memory's full rate beside the expanded values.
//
// Warps: RT softmax warpgroups (thread = row = TMEM lane), one that expands V, one with the TMA warp and the MMA warp. A unit is a
// (key tile, row tile); scores of unit u + 2 are issued behind P V of unit u into the same columns, so the softmax of one row tile
// runs beside the MMAs of the other (with a single row tile: of the next key tile, in the other score buffer).
#include "kv8_dev.cuh"
#include "tmap.cuh"

namespace lb {
namespace {

constexpr float P_OFFSET = 7.f, P_SLACK = 8.f;      // P relative to the reference times 2^7, at most 2^15; the reference moves by more than 2^8

struct PromptArgs {
  Kv8Cache c;
  Kv8Seqs s;
  Kv8Attn a;
  int n_splits;
  float scale_log2, cap_k;
  float* part;               // [T][Hq][n_splits][dv + 2], or nullptr
};

template <int KH, int MT>
struct PCfg {
  static constexpr int RT = (KH == 1 && MT == 1) ? 2 : 1;
  static constexpr int THREADS = (RT + 2) * 128;
  static constexpr int Q_BYTES = RT * 2 * KH * 16384;
  static constexpr int K_BYTES = KH * 16384, V8_BYTES = MT * 16384, V16_BYTES = MT * 32768;
  static constexpr int KS = 2, V8S = MT == 1 ? 2 : 1, V16S = MT == 1 ? 2 : 1;
  // registers of a softmax thread and of the others: together what the launch has (512 x 128 or 384 x 168)
  static constexpr int REGS_ROW = RT == 2 ? 184 : 232, REGS_REST = RT == 2 ? 72 : 136;
  static_assert(RT * 128 * REGS_ROW + 256 * REGS_REST <= (RT == 2 ? 512 * 128 : 384 * 168), "registers");
  static constexpr int TAIL = 1280 + RT * 512 + MT * 512;
  static constexpr int SMEM = Q_BYTES + KS * K_BYTES + V8S * V8_BYTES + V16S * V16_BYTES + TAIL;
  static constexpr int O_COL = 256;      // score buffers at 0 and 128
  static_assert(SMEM <= 227 * 1024 && O_COL + RT * MT * 128 <= 512, "sizes");
};

__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n"
      ::"r"(d_tmem), "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tm_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]),
      "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tm_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// packed fp32 pairs and the three-input maximum
__device__ __forceinline__ uint64_t f2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void f2_out(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <bool MASK, bool CAP, bool WIDE>
__device__ __forceinline__ void part_row(const uint32_t (&r)[32], const float4* sc, float fq, float ref, float cap_scale, int lo, int hi,
                                         uint32_t* w, float& mx0, float& mx1, float& total) {
  constexpr int PER = WIDE ? 32 : 8;
#pragma unroll
  for (int e = 0; e < 32; e += PER) {
    const float4 f = sc[e / 8];
    const float mul = fq * f.x, add = CAP ? f.y + ref + 0.5f * cap_scale : f.y + ref;
    const uint64_t mul2 = f2(mul, mul), add2 = f2(add, add);
    uint64_t acc = f2(0.f, 0.f);
#pragma unroll
    for (int j = e; j < e + PER; j += 2) {
      float z0, z1;
      if constexpr (CAP) {
        z0 = fmaf(softcap_r(__uint_as_float(r[j]) * mul, 1.f), cap_scale, add);
        z1 = fmaf(softcap_r(__uint_as_float(r[j + 1]) * mul, 1.f), cap_scale, add);
      } else {
        f2_out(f2_fma(f2(__uint_as_float(r[j]), __uint_as_float(r[j + 1])), mul2, add2), z0, z1);
      }
      if constexpr (MASK) {
        if (j < lo || j >= hi) z0 = -INFINITY;
        if (j + 1 < lo || j + 1 >= hi) z1 = -INFINITY;
      }
      if (j & 2) mx1 = fmax3(mx1, z0, z1);
      else mx0 = fmax3(mx0, z0, z1);
      const float y0 = ex2(z0), y1 = ex2(z1);
      acc = f2_add(acc, f2(y0, y1));
      w[j / 2] = half2_of(y0, y1);
    }
    float a0, a1;
    f2_out(acc, a0, a1);
    total = fmaf(a0 + a1, f.z, total);
  }
}

// One row of a tile: w = halves of 2^(z + ref), their sum with every value scale divided out, and the largest z + ref. WIDE: a
// scale for 32 keys or more, else for 8. MASK: keys outside [lo, hi) of the tile count nothing.
template <bool MASK, bool CAP, bool WIDE>
__device__ __forceinline__ void row_of_tile(uint32_t my_S, const float4* sc, float fq, float ref, float cap_scale, int lo, int hi,
                                            uint32_t (&w)[64], float& top, float& total) {
  float mx0 = -INFINITY, mx1 = -INFINITY;
  total = 0.f;
  uint32_t r[2][32];
  tmem_ld32(my_S, r[0]);
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    tmem_ld_wait();
    if (g < 3) tmem_ld32(my_S + g * 32 + 32, r[(g + 1) & 1]);      // on its way while this one is worked on
    part_row<MASK, CAP, WIDE>(r[g & 1], sc + g * 4, fq, ref, cap_scale, lo - g * 32, hi - g * 32, w + g * 16, mx0, mx1, total);
  }
  top = fmaxf(mx0, mx1);
}

// Writes NaN over a row's results in the columns in which one of its keys [lo, hi) has a NaN value. `first`: the first such key of each
// column. Where that lies in front of the row's window, the codes of the window are looked through. (Not inlined: it runs rarely, and
// inside the loop that writes the results it cost every launch 3%.)
__device__ __noinline__ void nan_columns(const Kv8Cache& c, const int* table, int kvh, const int* first, int lo, int hi, float* part,
                                         uint16_t* out) {
#pragma unroll 1
  for (int d = 0; d < c.dv; d += 16) {
    uint32_t seen = 0, look = 0;
#pragma unroll 1
    for (int j = 0; j < 16; ++j) {
      const int f = first[d + j];
      if (f < lo) look |= 1u << j;
      else if (f < hi) seen |= 1u << j;
    }
#pragma unroll 1
    for (int tok = lo; tok < hi && look; ++tok) {
      const int blk = table[tok / c.page];
      if (unsigned(blk) >= unsigned(c.n_blocks)) continue;
      const uint4 u = *reinterpret_cast<const uint4*>(c.v + ((long(blk) * c.Hkv + kvh) * c.page + tok % c.page) * c.dv + d);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
      uint32_t found = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t m = (w[k] & 0x7f7f7f7fu) + 0x01010101u;
        found |= ((m >> 7 & 1u) | (m >> 14 & 2u) | (m >> 21 & 4u) | (m >> 28 & 8u)) << (4 * k);
      }
      seen |= found & look;
      look &= ~found;
    }
    for (; seen; seen &= seen - 1) {
      const int at = d + __ffs(seen) - 1;
      if (part) part[at] = __uint_as_float(0x7fc00000u);
      else out[at] = 0x7fc0u;
    }
  }
}

template <int KH, int MT, bool CAP, bool WIDE>
__global__ void __launch_bounds__(PCfg<KH, MT>::THREADS, 1)
kv8_prompt_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ PromptArgs p) {
  using C = PCfg<KH, MT>;
  constexpr int RT = C::RT, KS = C::KS, V8S = C::V8S, V16S = C::V16S, BKV = 128;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {       // swizzled tiles; uniform per CTA, before any barrier
    if (threadIdx.x == 0) atomicCAS(p.s.status, 0, ST_BAD_ARGS);
    return;
  }
  uint8_t* q_s = smem;                                  // [RT][hi, lo][KH][128 rows x 128 bytes]
  uint8_t* k_s = q_s + C::Q_BYTES;
  uint8_t* v8_s = k_s + KS * C::K_BYTES;
  uint8_t* v16_s = v8_s + V8S * C::V8_BYTES;            // halves: [2 MT][128 keys x 128 bytes]
  uint64_t* bars = reinterpret_cast<uint64_t*>(v16_s + V16S * C::V16_BYTES);
  uint64_t* q_full = bars;
  uint64_t* k_full = bars + 1;      // [2]
  uint64_t* k_empty = bars + 3;     // [2]
  uint64_t* v8_full = bars + 5;     // [2]
  uint64_t* v8_empty = bars + 7;    // [2]
  uint64_t* v16_full = bars + 9;    // [2]
  uint64_t* v16_empty = bars + 11;  // [2]
  uint64_t* s_full = bars + 13;     // [2]
  uint64_t* p_ready = bars + 15;    // [2]
  uint64_t* o_done = bars + 17;     // [2]
  uint64_t* sc_full = bars + 19;    // [4]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 23);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* s_nan = reinterpret_cast<int*>(bars + 24);       // first and last key with a NaN value
  float4* s_sc = reinterpret_cast<float4*>(bars + 32);  // [4][16]: key scale, log2 of the value scale 2^e, 2^-e, per 8 keys
  float* s_q = reinterpret_cast<float*>(bars + 160);    // [RT * 128]: a row's power of two times the score scale
  int* s_first = reinterpret_cast<int*>(s_q + RT * 128);      // [MT * 128]: a column's first key with a NaN value

  const Kv8Cache& c = p.c;
  const int G = p.a.Hq / c.Hkv;
  const int kvh = blockIdx.y % c.Hkv, split = blockIdx.y / c.Hkv, seq = blockIdx.z;
  const int q0 = p.s.cu[seq], n_new = p.s.cu[seq + 1] - q0;
  // tiles are handed out from the last to the first: the last sees the most keys
  const int row0 = (int(gridDim.x) - 1 - int(blockIdx.x)) * (RT * 128);
  if (n_new <= 0 || row0 >= n_new * G) return;
  const int ctx = max(p.s.ctx[seq], 0);
  if (q0 < 0 || long(q0) + n_new > p.s.T || n_new > p.s.max_new || ctx > long(p.s.width) * c.page) {
    if (threadIdx.x == 0) atomicCAS(p.s.status, 0, ST_BAD_ARGS);
    return;
  }
  const int rows = min(RT * 128, n_new * G - row0);
  const int n_rt = rows > 128 ? 2 : 1;
  const int pos_first = ctx - n_new + row0 / G, pos_last = ctx - n_new + (row0 + rows - 1) / G;
  const int key_hi = min(ctx, pos_last + 1);
  const int key_lo = p.a.window > 0 ? max(0, pos_first - p.a.window + 1) : 0;
  const int tile_a = key_lo / BKV, tiles_all = max(0, (key_hi + BKV - 1) / BKV - tile_a);
  const int per = (tiles_all + p.n_splits - 1) / p.n_splits;
  const int tile0 = tile_a + split * per, n_tiles = max(0, min(tiles_all - split * per, per));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int D = c.dv;
  const int wg = warp >> 2;                             // < RT: softmax, RT: values, RT + 1: TMA and MMA

  if (threadIdx.x == 0) {
    mbar_init(q_full, (RT + 1) * 128);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v8_full[i], 1);
      mbar_init(&v8_empty[i], 128);
      mbar_init(&v16_full[i], 128);
      mbar_init(&v16_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 128);
      mbar_init(&o_done[i], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&sc_full[i], 32);
    *abort_flag = 0;
    s_nan[0] = 0x7fffffff;
    s_nan[1] = -1;
    mbar_fence_init();
  }
  for (int i = threadIdx.x; i < MT * 128; i += C::THREADS) s_first[i] = 0x7fffffff;
  if (warp == (RT + 1) * 4) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto fail = [&](int code) { *abort_flag = 1; atomicCAS(p.s.status, 0, code | SITE_PREFILL_ATTN); return false; };

  // Queries, by the softmax and the value warps, a row at a time: a power of two, two e4m3 terms. Not finite: a NaN code. Eight rows
  // are fetched at once: a fetch behind another row's stores waits for them, and 22 rows in a chain took 12 us.
  if (wg <= RT) {
    constexpr int DIMS = KH * 4, NW = (RT + 1) * 4, ROWS = 8;      // columns of a lane, warps, rows in flight
    const int d = lane * DIMS, ch = d / 16;
#pragma unroll 1
    for (int r0 = warp; r0 < RT * 128; r0 += NW * ROWS) {
      uint32_t u[ROWS][KH * 2];
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int r = r0 + i * NW, gr = row0 + r;
#pragma unroll
        for (int k = 0; k < KH * 2; ++k) u[i][k] = 0u;
        if (r < rows && d < c.dk) {
          const int tok = gr / G;
          const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(p.a.q) + (long(q0) + tok) * p.a.q_tok + (kvh * G + gr - tok * G) * p.a.q_head + d;
          if ((reinterpret_cast<uintptr_t>(src) & (KH * 8 - 1)) == 0) {
            if (KH == 1) *reinterpret_cast<uint2*>(u[i]) = *reinterpret_cast<const uint2*>(src);
            else *reinterpret_cast<uint4*>(u[i]) = *reinterpret_cast<const uint4*>(src);
          } else {
            const uint16_t* h = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
            for (int k = 0; k < KH * 2; ++k) u[i][k] = h[2 * k] | uint32_t(h[2 * k + 1]) << 16;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int r = r0 + i * NW;
        if (r >= RT * 128) break;
        uint32_t m = 0;
#pragma unroll
        for (int k = 0; k < KH * 2; ++k) {
          const uint32_t lo = u[i][k] & 0x7fffu, hi = (u[i][k] >> 16) & 0x7fffu;
          m = max(m, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
        }
        m = __reduce_max_sync(0xffffffffu, m);
        const float qs = kv8_scale_of(__uint_as_float(m << 16)), inv = kv8_inverse(qs);
        if (lane == 0) s_q[r] = qs * (CAP ? p.cap_k : p.scale_log2);
        uint32_t hi4[KH], lo4[KH];
#pragma unroll
        for (int k = 0; k < KH * 2; ++k) {
          const float a0 = __uint_as_float(u[i][k] << 16) * inv, a1 = __uint_as_float(u[i][k] & 0xffff0000u) * inv;
          uint32_t hh = e4m3x2(a0, a1);
          if ((u[i][k] & 0x7f80u) == 0x7f80u) hh |= 0x7fu;
          if ((u[i][k] & 0x7f800000u) == 0x7f800000u) hh |= 0x7f00u;
          const float2 f = __half22float2(e4m3x2_to_half2(hh));
          // the remainder in the units of the first term: its lower end, 2^-10 of a largest code of 128 or more, is 2^-17 of the
          // row's largest value; bf16 values that small have a step of 2^-9 of themselves
          const uint32_t ll = e4m3x2(a0 - f.x, a1 - f.y);
          if (k & 1) { hi4[k / 2] |= hh << 16; lo4[k / 2] |= ll << 16; }
          else { hi4[k / 2] = hh; lo4[k / 2] = ll; }
        }
        uint8_t* dst = q_s + ((r / 128) * 2 * KH + ch / 8) * 16384 + (r % 128) * 128 + (((ch & 7) ^ (r & 7)) << 4) + d % 16;
        if (KH == 1) {
          *reinterpret_cast<uint32_t*>(dst) = hi4[0];
          *reinterpret_cast<uint32_t*>(dst + KH * 16384) = lo4[0];
        } else {
          *reinterpret_cast<uint2*>(dst) = make_uint2(hi4[0], hi4[KH - 1]);
          *reinterpret_cast<uint2*>(dst + KH * 16384) = make_uint2(lo4[0], lo4[KH - 1]);
        }
      }
    }
    fence_proxy_async_smem();
    mbar_arrive(q_full);
  }
  if (wg == RT + 1) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS_REST));
    if (warp == (RT + 1) * 4 + 1) {
      // ---------------------------------------------------------------- TMA: the lanes fetch table and scales, lane 0 issues
      const int* bt = p.s.table + seq * p.s.ld_table;
      const int ppb = BKV / c.page, tiles_per_fill = 32 / ppb;
      int pg_reg = 0;
      float ks_reg = 0.f, vs_reg = 0.f;
      bool ok = true;
      for (int i = 0; ok && i < n_tiles; ++i) {
        const int at = i % tiles_per_fill;
        if (at == 0) {
          const long page = long(tile0 + i) * ppb + lane;
          pg_reg = page * c.page < ctx ? bt[page] : c.n_blocks;      // (a block outside the cache reads as zeros)
          ks_reg = vs_reg = 0.f;
          if (unsigned(pg_reg) < unsigned(c.n_blocks)) {
            const long u = long(pg_reg) * c.Hkv + kvh;
            ks_reg = c.k_scale[u];
            vs_reg = c.v_scale[u];
          } else {
            if (page * c.page < key_hi && page * c.page + c.page > key_lo) atomicCAS(p.s.status, 0, ST_BAD_ARGS);
            pg_reg = c.n_blocks;
          }
        }
        const int ks = i % KS, v8 = i % V8S;
        if (i >= KS && !__all_sync(0xffffffffu, mbar_wait(&k_empty[ks], ((i / KS) - 1) & 1, abort_flag))) {
          if (lane == 0) fail(ST_TIMEOUT_EMPTY);
          break;
        }
        // slot i % 4 held tile i - 4: its softmax is over, since the scores of tile i - 2 are done (k_empty) and stand behind it
        {
          const int g = at * ppb + (lane & 15) * 8 / c.page;
          const float a = __shfl_sync(0xffffffffu, ks_reg, g), b = __shfl_sync(0xffffffffu, vs_reg, g);
          const int ev = kv8_log2(kv8_value_scale(b));
          if (lane < 16) s_sc[(i & 3) * 16 + lane] = make_float4(a, float(ev), __uint_as_float(uint32_t(127 - ev) << 23), 0.f);
          mbar_arrive(&sc_full[i & 3]);
        }
        if (lane == 0) mbar_expect_tx(&k_full[ks], C::K_BYTES);
        for (int g = 0; g < ppb; ++g) {
          const int pg = __shfl_sync(0xffffffffu, pg_reg, at * ppb + g);
          if (lane == 0)
            for (int h = 0; h < KH; ++h)
              tma_load_2d(k_s + ks * C::K_BYTES + h * 16384 + g * c.page * 128, &tmK, &k_full[ks], h * 128, (pg * c.Hkv + kvh) * c.page);
        }
        if (i >= V8S && !__all_sync(0xffffffffu, mbar_wait(&v8_empty[v8], ((i / V8S) - 1) & 1, abort_flag))) {
          if (lane == 0) fail(ST_TIMEOUT_EMPTY);
          break;
        }
        if (lane == 0) mbar_expect_tx(&v8_full[v8], C::V8_BYTES);
        for (int g = 0; g < ppb; ++g) {
          const int pg = __shfl_sync(0xffffffffu, pg_reg, at * ppb + g);
          if (lane == 0)
            for (int h = 0; h < MT; ++h)
              tma_load_2d(v8_s + v8 * C::V8_BYTES + h * 16384 + g * c.page * 128, &tmV, &v8_full[v8], h * 128, (pg * c.Hkv + kvh) * c.page);
        }
      }
    } else if (warp == (RT + 1) * 4 && lane == 0 && n_tiles > 0) {
      // ---------------------------------------------------------------- MMA
      constexpr uint32_t idesc_s = umma_idesc(128, BKV, 0, 0, 0, 0);            // e4m3 x e4m3
      constexpr uint32_t idesc_o = umma_idesc(128, MT * 128, 0, 0, 0, 1);       // half x half, V is MN-major
      // descriptors are made once; a step adds its offset in 16-byte units (made anew for every MMA they took the issuing thread
      // twice as long as the MMAs)
      const uint64_t dq = umma_desc_k_sw128(smem_u32(q_s)), dk = umma_desc_k_sw128(smem_u32(k_s));
      const uint64_t dv = umma_desc_mn_sw128(smem_u32(v16_s), 16384, 1024);
      const int units = n_tiles * n_rt;
      auto issue_s = [&](int u) -> bool {
        const int i = u / n_rt, r = u % n_rt, st = i % KS;
        if (!mbar_wait(&k_full[st], (i / KS) & 1, abort_flag)) return fail(ST_TIMEOUT_FULL);
        tc_fence_after();
        const uint64_t da = dq + uint32_t(r) * (2 * KH * 1024), db = dk + uint32_t(st) * (C::K_BYTES / 16);
        const uint32_t ts = tmem + (u & 1) * 128;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int h = 0; h < KH; ++h) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_f8(ts, da + ((t * KH + h) * 1024 + k * 2), db + (h * 1024 + k * 2), idesc_s, (t | h | k) ? 1u : 0u);
          }
        }
        umma_commit(&s_full[u & 1]);
        if (r == n_rt - 1) umma_commit(&k_empty[st]);
        return true;
      };
      bool ok = mbar_wait(q_full, 0, abort_flag) || fail(ST_TIMEOUT_FULL);
      ok = ok && issue_s(0);
      if (ok && units > 1) ok = issue_s(1);
      for (int u = 0; ok && u < units; ++u) {
        const int i = u / n_rt, r = u % n_rt, st = i % V16S;
        if (!mbar_wait(&v16_full[st], (i / V16S) & 1, abort_flag)) { fail(ST_TIMEOUT_FULL); break; }
        if (!mbar_wait(&p_ready[u & 1], (u >> 1) & 1, abort_flag)) { fail(ST_TIMEOUT_FLAG); break; }
        tc_fence_after();
        const uint64_t db = dv + uint32_t(st) * (C::V16_BYTES / 16);
        const uint32_t to = tmem + C::O_COL + r * (MT * 128), ta = tmem + (u & 1) * 128;
#pragma unroll
        for (int k = 0; k < BKV / 16; ++k) umma_f16_ts(to, ta + k * 8, db + k * 128, idesc_o, (i | k) ? 1u : 0u);
        umma_commit(&o_done[u & 1]);
        if (r == n_rt - 1) umma_commit(&v16_empty[st]);
        if (u + 2 < units && !issue_s(u + 2)) break;
      }
    }
  } else if (wg == RT) {
    // ------------------------------------------------------------------ values: e4m3 -> half, thread = key
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS_REST));
    const int key = threadIdx.x - RT * 128;
    bool ok = true;
    for (int i = 0; i < n_tiles; ++i) {
      const int v8 = i % V8S, v16 = i % V16S;
      ok = ok && __all_sync(0xffffffffu, mbar_wait(&v8_full[v8], (i / V8S) & 1, abort_flag));
      if (ok && i >= V16S) ok = __all_sync(0xffffffffu, mbar_wait(&v16_empty[v16], ((i / V16S) - 1) & 1, abort_flag));
      if (!ok) {
        if (lane == 0) fail(ST_TIMEOUT_FULL);
        break;
      }
      const int tok = (tile0 + i) * BKV + key;
      const bool seen = tok >= key_lo && tok < key_hi;      // the others may hold anything: zeros
      const uint8_t* src = v8_s + v8 * C::V8_BYTES + key * 128;
      uint8_t* dst = v16_s + v16 * C::V16_BYTES + key * 128;
#pragma unroll 1
      for (int h = 0; h < MT; ++h) {
        uint32_t x[32];
        uint32_t any = 0;
#pragma unroll
        for (int ch = 0; ch < 8; ++ch) {
          uint4 w = make_uint4(0u, 0u, 0u, 0u);
          if (seen) w = *reinterpret_cast<const uint4*>(src + h * 16384 + ((ch ^ (key & 7)) << 4));
          x[4 * ch] = w.x; x[4 * ch + 1] = w.y; x[4 * ch + 2] = w.z; x[4 * ch + 3] = w.w;
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) any |= (x[j] & 0x7f7f7f7fu) + 0x01010101u;
        if (any & 0x80808080u) {
          // NaN codes: noted (at the end, rows become NaN in the columns of those they see), and not multiplied with the zeros of
          // rows that do not
          atomicMin(&s_nan[0], tok);
          atomicMax(&s_nan[1], tok);
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            for (int e = 0; e < 4; ++e) {
              if (((x[j] >> (8 * e)) & 0x7fu) == 0x7fu) {
                atomicMin(&s_first[h * 128 + 4 * j + e], tok);
                x[j] &= ~(0xffu << (8 * e));
              }
            }
          }
        }
#pragma unroll
        for (int ch = 0; ch < 8; ++ch) {
          uint32_t o[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const __half2 y = e4m3x2_to_half2(x[4 * ch + j / 2] >> (16 * (j & 1)));
            o[j] = *reinterpret_cast<const uint32_t*>(&y);
          }
          uint8_t* d8 = dst + (h * 2 + ch / 4) * 16384;
          const int c0 = (ch % 4) * 2;
          *reinterpret_cast<uint4*>(d8 + ((c0 ^ (key & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4*>(d8 + (((c0 + 1) ^ (key & 7)) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
        }
      }
      mbar_arrive(&v8_empty[v8]);
      fence_proxy_async_smem();
      mbar_arrive(&v16_full[v16]);
    }
  } else {
    // ------------------------------------------------------------------ softmax, thread = row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REGS_ROW));
    const int row = threadIdx.x & 127;
    const int gr = row0 + wg * 128 + row;
    const bool row_ok = wg * 128 + row < rows;
    const int tok_row = gr / G, head = kvh * G + gr % G;
    const long t = long(q0) + tok_row;
    const int pos = ctx - n_new + tok_row;
    const uint32_t lane_off = uint32_t((warp & 3) * 32) << 16;
    bool ok = __all_sync(0xffffffffu, mbar_wait(q_full, 0, abort_flag));
    if (!ok) fail(ST_TIMEOUT_FULL);
    const float fq = s_q[wg * 128 + row];
    const int hi = row_ok ? min(ctx, pos + 1) : 0, lo = p.a.window > 0 ? max(0, pos - p.a.window + 1) : 0;
    const uint32_t my_O = tmem + C::O_COL + wg * (MT * 128) + lane_off;
    float m = -INFINITY, l = 0.f;
    if (ok && wg < n_rt) {
      for (int i = 0; i < n_tiles; ++i) {
        const int u = i * n_rt + wg, b = u & 1;
        ok = __all_sync(0xffffffffu, mbar_wait(&sc_full[i & 3], (i >> 2) & 1, abort_flag)) &&
             __all_sync(0xffffffffu, mbar_wait(&s_full[b], (u >> 1) & 1, abort_flag));
        if (!ok) {
          fail(ST_TIMEOUT_TMEM_FULL);
          break;
        }
        tc_fence_after();
        const uint32_t my_S = tmem + b * 128 + lane_off;
        const float4* sc = s_sc + (i & 3) * 16;
        const int key0 = (tile0 + i) * BKV;
        // entirely visible to every row of the CTA: no masks
        const bool full = rows == RT * 128 && key0 + BKV <= min(ctx, pos_first + 1) && (p.a.window == 0 || key0 > pos_last - p.a.window);
        // With the reference as it stands; where a row's largest passes it by more than the slack (in the first tile, and rarely
        // after it), the references move, O and l follow, and the tile is taken again: its scores are still there.
        uint32_t w[64];
        float top, total;
#pragma unroll 1
        for (int again = 0;; ++again) {
          const float ref = m == -INFINITY ? 0.f : P_OFFSET - m;
          if (full) row_of_tile<false, CAP, WIDE>(my_S, sc, fq, ref, p.scale_log2, 0, 0, w, top, total);
          else row_of_tile<true, CAP, WIDE>(my_S, sc, fq, ref, p.scale_log2, lo - key0, hi - key0, w, top, total);
          const bool over = m == -INFINITY ? top > -INFINITY : top > P_OFFSET + P_SLACK;
          if (again || !__any_sync(0xffffffffu, over)) break;
          float alpha = 1.f;
          if (over) {
            const float now = top - ref;
            alpha = ex2(m - now);                  // (0 at first)
            m = now;
          }
          l *= alpha;
          if (i > 0) {
            // O may be touched once P V of the tile before is done: with two row tiles it ran before these scores, with one it may
            // not have
            if (n_rt == 1 && !__all_sync(0xffffffffu, mbar_wait(&o_done[(u - 1) & 1], ((u - 1) >> 1) & 1, abort_flag))) {
              ok = fail(ST_TIMEOUT_TMEM_EMPTY);
              break;
            }
            tc_fence_after();
#pragma unroll 1
            for (int d = 0; d < MT * 128; d += 32) {
              uint32_t r[32];
              tmem_ld32(my_O + d, r);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * alpha);
              tm_st32(my_O + d, r);
            }
          }
        }
        if (!ok) break;
        tm_st32(my_S, *reinterpret_cast<uint32_t(*)[32]>(w));
        tm_st32(my_S + 32, *reinterpret_cast<uint32_t(*)[32]>(w + 32));
        l += total;                                // (once per tile: thousands of single additions would cost it 2^-20)
        tm_st_wait();
        tc_fence_before();
        mbar_arrive(&p_ready[b]);
      }
    }
    if (ok && wg < n_rt && n_tiles > 0) {
      const int u = (n_tiles - 1) * n_rt + wg;
      if (!__all_sync(0xffffffffu, mbar_wait(&o_done[u & 1], (u >> 1) & 1, abort_flag))) ok = fail(ST_TIMEOUT_TMEM_FULL);
    }
    if (ok && wg < n_rt) {
      tc_fence_after();
      float top = m == -INFINITY ? m : m - P_OFFSET, den = l, inv = 0.f;
      float* part = p.part ? p.part + ((t * p.a.Hq + head) * p.n_splits + split) * (D + 2) : nullptr;
      if (part) {
        if (row_ok) {
          part[D] = top;
          part[D + 1] = l;
        }
      } else {
        if (p.a.sink) {
          const float f = kv8_add_sink((row_ok ? p.a.sink[head] : 0.f) * 1.4426950408889634f, top, den);
          inv = den > 0.f || den != den ? f / den : 0.f;
        } else {
          inv = den > 0.f || den != den ? 1.f / den : 0.f;
        }
        if (p.a.lse && row_ok) p.a.lse[t * p.a.Hq + head] = den > 0.f ? top + log2f(den) : -INFINITY;
      }
#pragma unroll 1
      for (int d = 0; d < MT * 128; d += 32) {
        uint32_t r[32];
        if (n_tiles > 0) {
          tmem_ld32(my_O + d, r);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) r[j] = 0u;
        }
        if (!row_ok || d >= D) continue;
        if (part) {
#pragma unroll
          for (int j = 0; j < 32; j += 2)
            if (d + j < D) *reinterpret_cast<float2*>(part + d + j) = make_float2(__uint_as_float(r[j]), __uint_as_float(r[j + 1]));
        } else {
          __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.a.out) + t * p.a.o_tok + long(head) * D + d;
          uint32_t w[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) w[j] = pack_bf16x2(__uint_as_float(r[2 * j]) * inv, __uint_as_float(r[2 * j + 1]) * inv);
          if ((reinterpret_cast<uintptr_t>(o) & 15) == 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (d + 8 * j < D) reinterpret_cast<uint4*>(o)[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (d + j < D) reinterpret_cast<uint16_t*>(o)[j] = uint16_t(w[j / 2] >> (16 * (j & 1)));
          }
        }
      }
      if (row_ok && s_nan[1] >= lo && s_nan[0] < hi)
        nan_columns(c, p.s.table + seq * p.s.ld_table, kvh, s_first, lo, min(hi, s_nan[1] + 1), part,
                    static_cast<uint16_t*>(p.a.out) + t * p.a.o_tok + long(head) * D);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == (RT + 1) * 4) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int KH, int MT, bool CAP, bool WIDE>
cudaError_t launch(const CUtensorMap* tk, const CUtensorMap* tv, const PromptArgs& p, cudaStream_t st) {
  using C = PCfg<KH, MT>;
  auto kfn = kv8_prompt_kernel<KH, MT, CAP, WIDE>;
  static DeviceOnce once;
  const cudaError_t e = once.shared_memory(reinterpret_cast<const void*>(kfn), C::SMEM);
  if (e != cudaSuccess) return e;
  const long rows = long(p.s.max_new) * (p.a.Hq / p.c.Hkv);
  const dim3 grid(unsigned((rows + C::RT * 128 - 1) / (C::RT * 128)), p.c.Hkv * p.n_splits, p.s.n);
  kfn<<<grid, C::THREADS, C::SMEM, st>>>(*tk, *tv, p);
  return cudaGetLastError();
}

}  // namespace

int kv8_prompt_launch(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Attn& a, int n_splits, float* part, cudaStream_t st) {
  if (s.n <= 0 || s.T <= 0 || s.max_new <= 0) return 0;
  const uint64_t rows = uint64_t(c.n_blocks) * c.Hkv * c.page;
  const CUtensorMap* tk = tmap_2d(c.k, rows, c.dk, c.dk, c.page, 128, TM_U8, true);
  const CUtensorMap* tv = tmap_2d(c.v, rows, c.dv, c.dv, c.page, 128, TM_U8, true);
  if (!tk || !tv) {
    kv8_set_error(tmap_last_error());
    return 1;
  }
  PromptArgs p{c, s, a, n_splits, a.scale * 1.4426950408889634f, 0.f, n_splits > 1 ? part : nullptr};
  const bool cap = a.softcap > 0.f;
  if (cap) {
    p.cap_k = 2.f * 1.4426950408889634f * a.scale / a.softcap;
    p.scale_log2 = 2.f * 1.4426950408889634f * a.softcap;
  }
  const int kh = (c.dk + 127) / 128, mt = (c.dv + 127) / 128;
  cudaError_t e = cudaErrorInvalidValue;
  const bool wide = c.page >= 32;
#define LB_KV8(K_, V_)                                                                                                          \
  if (kh == K_ && mt == V_)                                                                                                     \
    e = cap ? (wide ? launch<K_, V_, true, true>(tk, tv, p, st) : launch<K_, V_, true, false>(tk, tv, p, st))                   \
            : (wide ? launch<K_, V_, false, true>(tk, tv, p, st) : launch<K_, V_, false, false>(tk, tv, p, st));
  LB_KV8(1, 1) LB_KV8(1, 2) LB_KV8(2, 1) LB_KV8(2, 2)
#undef LB_KV8
  if (e == cudaSuccess && n_splits > 1) e = kv8_join(c, s, a, n_splits, part, st);
  if (e != cudaSuccess) kv8_set_error(cudaGetErrorString(e));
  return e != cudaSuccess;
}

}  // namespace lb
