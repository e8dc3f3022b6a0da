// Sums of attention weights per key of the 8-bit cache, for eviction: w[key] += sum over rows and query heads of
// exp(score - lse), with the log-sum-exp of every row and head from the attention itself.
//
// Decode: the attention kernel leaves its scores (4 bytes a head and key, an eighth of the keys' own bytes at 4 to 8 heads of 128
// per kv head, where scores made anew would read all keys again), and kv8_score_sums_kernel adds them up,
// four keys to a thread so that their loads fly together (64 sequences of 750 to 2250 keys: 8 us alone, 17 with one key and a
// shared copy of the log-sum-exps).
//
// Rows of a prompt: the scores once more. kv8_queries_kernel packs the rows that count, 64 (token, head) rows of a kv head to a
// record: their two e4m3 terms in the layout that the MMA reads, powers of two, log-sum-exps and positions. kv8_weights_kernel,
// a CTA per 256 keys of a kv head, keeps its two key tiles in shared memory and streams the records past them:
// S^T[128 keys, 64 rows] = K . Q^T on tcgen05, with the terms, scales and order of the attention, whose sums its scores have to be
// bit for bit: the tensor cores cut off what does not fit a sum, and scores summed in another order gave weights 10^-6 too large.
// A thread has a key and adds up its columns over all records, so nothing crosses threads and the result does not depend on any
// order but the rows' own; what the additions of records round off is carried along (single additions of 0.88 from 20800 rows ended 5e-5
// off, where all of them round the same way; it costs nothing that can be measured). Two score tiles are made ahead of their use. 64 exponentials per key and record
// and the records' traffic bound it: 64 rows of 32 heads over 16K keys add 30 us to the call, all 1024 rows 295 (a mask branch per
// score instead of per record and one score tile: 57 and 510).
#include <type_traits>
#include "kv8_dev.cuh"
#include "tmap.cuh"

namespace lb {
namespace {

constexpr int RN = 64, BKV = 128;
constexpr int SUM_THREADS = 128, SUM_KEYS = 4;      // of kv8_score_sums_kernel: keys of a thread lie SUM_THREADS apart
constexpr int HEAD = 1024;               // of a record: powers of two [64], log-sum-exps [64], positions [64]; behind it the first, then the second terms

struct WeightArgs {
  Kv8Cache c;
  Kv8Seqs s;
  Kv8Attn a;
  int observe, max_rt;            // last rows of a sequence that count (0: all); records of a sequence and head at most
  long per_head;                  // records that a kv head has room for
  int packed;                     // they lie in the order of the call's rows; else max_rt to a sequence
  float scale_log2, cap_k;
  float* w; long w_seq, w_head; int w_keys;
  uint8_t* records;
};

// Rows of a sequence that count: the first, how many (token, head) rows, position of the first, length
struct Rows {
  int first, rows, base, ctx, q0;
};
__device__ __forceinline__ Rows rows_of(const WeightArgs& p, int seq, int G) {
  Rows r;
  r.q0 = p.s.cu[seq];
  const int n_new = p.s.cu[seq + 1] - r.q0;
  r.ctx = max(p.s.ctx[seq], 0);
  r.first = p.observe > 0 ? max(0, n_new - p.observe) : 0;
  r.base = r.ctx - n_new + r.first;
  r.rows = (n_new - r.first) * G;
  if (n_new <= 0 || r.q0 < 0 || long(r.q0) + n_new > p.s.T || n_new > p.s.max_new || r.ctx > p.w_keys ||
      r.ctx > long(p.s.width) * p.c.page) {
    if (threadIdx.x == 0 && n_new > 0) atomicCAS(p.s.status, 0, ST_BAD_ARGS);
    r.rows = 0;
  }
  return r;
}

// Index of a sequence's first record among its kv head's. In the order of the rows: a sequence of n rows has ceil(n G / 64) records at
// most, and floor(q0 G / 64) + sequence leaves it that many, up to ceil(T G / 64) + sequences in all.
__device__ __forceinline__ long first_record(const WeightArgs& p, int seq, int q0, int G) {
  return p.packed ? long(q0) * G / RN + seq : long(seq) * p.max_rt;
}

template <int KH>
__global__ void __launch_bounds__(256) kv8_queries_kernel(const WeightArgs p) {
  griddep_wait();
  griddep_launch();
  const int G = p.a.Hq / p.c.Hkv, kvh = blockIdx.y;
  int seq = blockIdx.z, rt = blockIdx.x;
  if (p.packed) {
    // the last sequence whose records begin here or before
    int lo = 0, hi = p.s.n;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (first_record(p, mid, p.s.cu[mid], G) <= long(blockIdx.x)) lo = mid + 1;
      else hi = mid;
    }
    if (lo == 0) return;
    seq = lo - 1;
    rt = int(blockIdx.x - first_record(p, seq, p.s.cu[seq], G));
  }
  const Rows x = rows_of(p, seq, G);
  if (long(rt) * RN >= x.rows) return;
  const int n = min(RN, x.rows - rt * RN);
  uint8_t* rec = p.records + (kvh * p.per_head + first_record(p, seq, x.q0, G) + rt) * (HEAD + 2 * KH * RN * 128);
  float* head = reinterpret_cast<float*>(rec);
  constexpr int PER = RN * KH * 8 / 256;                  // chunks of 16 values of a thread
#pragma unroll 1
  for (int j = 0; j < PER; ++j) {
    const int i = threadIdx.x + j * 256, r = i / (KH * 8), ch = i % (KH * 8);      // a row's chunks lie in neighbouring lanes
    uint32_t u[8];
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) u[k] = 0u;
    if (r < n && ch * 16 < p.c.dk) {
      const int gr = rt * RN + r;
      const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(p.a.q) + long(x.q0 + x.first + gr / G) * p.a.q_tok +
                                 (kvh * G + gr % G) * p.a.q_head + ch * 16;
      if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
        *reinterpret_cast<uint4*>(u) = reinterpret_cast<const uint4*>(src)[0];
        *reinterpret_cast<uint4*>(u + 4) = reinterpret_cast<const uint4*>(src)[1];
      } else {
        const uint16_t* hs = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
        for (int k = 0; k < 8; ++k) u[k] = hs[2 * k] | uint32_t(hs[2 * k + 1]) << 16;
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t lo = u[k] & 0x7fffu, hi = (u[k] >> 16) & 0x7fffu;
      m = max(m, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
    }
#pragma unroll
    for (int o = 1; o < KH * 8; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float qs = kv8_scale_of(__uint_as_float(m << 16)), inv = kv8_inverse(qs);
    if (ch == 0) {
      const int gr = rt * RN + r;
      float lse = INFINITY;                                // rows that see nothing or do not exist weigh nothing
      if (r < n) {
        lse = p.a.lse[long(x.q0 + x.first + gr / G) * p.a.Hq + kvh * G + gr % G];
        if (lse == -INFINITY) lse = INFINITY;
      }
      head[r] = qs * (p.a.softcap > 0.f ? p.cap_k : p.scale_log2);
      head[RN + r] = lse;
      reinterpret_cast<int*>(head)[2 * RN + r] = r < n ? x.base + gr / G : -1;
    }
    uint32_t hi4[4], lo4[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      hi4[k] = lo4[k] = 0u;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t v = u[2 * k + e];
        const float a0 = __uint_as_float(v << 16) * inv, a1 = __uint_as_float(v & 0xffff0000u) * inv;
        uint32_t hh = e4m3x2(a0, a1);
        if ((v & 0x7f80u) == 0x7f80u) hh |= 0x7fu;
        if ((v & 0x7f800000u) == 0x7f800000u) hh |= 0x7f00u;
        const float2 f = __half22float2(e4m3x2_to_half2(hh));
        hi4[k] |= hh << (16 * e);
        lo4[k] |= e4m3x2(a0 - f.x, a1 - f.y) << (16 * e);
      }
    }
    uint8_t* dst = rec + HEAD + (ch / 8) * (RN * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
    *reinterpret_cast<uint4*>(dst) = make_uint4(hi4[0], hi4[1], hi4[2], hi4[3]);
    *reinterpret_cast<uint4*>(dst + KH * RN * 128) = make_uint4(lo4[0], lo4[1], lo4[2], lo4[3]);
  }
}

template <int KH>
struct WCfg {
  static constexpr int K_BYTES = KH * 16384;              // two of them
  static constexpr int R_BYTES = HEAD + 2 * KH * RN * 128, ST = KH == 1 ? 4 : 3;      // records in flight
  static constexpr int TAIL = 256;
  static constexpr int SMEM = 2 * K_BYTES + ST * R_BYTES + TAIL + 1024;           // two CTAs to an SM at KH = 1
};

template <int KH, bool CAP>
__global__ void __launch_bounds__(320, KH == 1 ? 2 : 1) kv8_weights_kernel(const __grid_constant__ CUtensorMap tmK, const WeightArgs p) {
  using C = WCfg<KH>;
  constexpr int ST = C::ST;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* k_s = smem;
  uint8_t* r_s = k_s + 2 * C::K_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(r_s + ST * C::R_BYTES);
  uint64_t* k_full = bars;         // [2]
  uint64_t* r_full = bars + 2;     // [4]
  uint64_t* r_empty = bars + 6;    // [4]
  uint64_t* s_full = bars + 10;    // [2 tiles][2 buffers]
  uint64_t* s_empty = bars + 14;   // [2][2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 18);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const Kv8Cache& c = p.c;
  const int G = p.a.Hq / c.Hkv;
  const int kvh = blockIdx.y, seq = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  griddep_wait();
  griddep_launch();
  const Rows x = rows_of(p, seq, G);
  const int tile0 = blockIdx.x * 2, n_tiles = min(2, (x.ctx + BKV - 1) / BKV - tile0);
  if (x.ctx > long(gridDim.x) * 2 * BKV && threadIdx.x == 0) atomicCAS(p.s.status, 0, ST_BAD_ARGS);      // longer than announced
  if (x.rows <= 0 || n_tiles <= 0) return;
  // records whose rows see any of these keys: positions from key0 on, and no further behind the last key than the window
  const int key0 = tile0 * BKV, key1 = min(x.ctx, key0 + n_tiles * BKV) - 1;
  const int n_rt = (x.rows + RN - 1) / RN;
  const long r_lo = long(max(0, key0 - x.base)) * G;
  const int ra = int(min(long(n_rt), r_lo / RN));
  const int rb = p.a.window > 0 ? int(min(long(n_rt), max(0l, (long(key1) + p.a.window - x.base) * G + RN - 1) / RN)) : n_rt;
  if (ra >= rb) return;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) mbar_init(&k_full[i], 1);
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], 128);
    }
    for (int i = 0; i < ST; ++i) {
      mbar_init(&r_full[i], 1);
      mbar_init(&r_empty[i], 9);
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, 4 * RN);
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
    const long page = long(tile0) * ppb + lane;            // 2 ppb <= 32 pages
    int pg = page * c.page < x.ctx ? bt[page] : c.n_blocks;
    if (unsigned(pg) > unsigned(c.n_blocks)) pg = c.n_blocks;      // (reads as zeros; recorded with the scales)
    for (int t = 0; t < n_tiles; ++t) {
      if (lane == 0) mbar_expect_tx(&k_full[t], C::K_BYTES);
      for (int g = 0; g < ppb; ++g) {
        const int b = __shfl_sync(0xffffffffu, pg, t * ppb + g);
        if (lane == 0)
          for (int h = 0; h < KH; ++h)
            tma_load_2d(k_s + t * C::K_BYTES + h * 16384 + g * c.page * 128, &tmK, &k_full[t], h * 128, (b * c.Hkv + kvh) * c.page);
      }
    }
    const uint8_t* rec = p.records + (kvh * p.per_head + first_record(p, seq, x.q0, G)) * C::R_BYTES;
    for (int i = 0; i < rb - ra; ++i) {
      const int st = i % ST;
      if (i >= ST && !__all_sync(0xffffffffu, mbar_wait(&r_empty[st], ((i / ST) - 1) & 1, abort_flag))) {
        if (lane == 0) fail(ST_TIMEOUT_EMPTY);
        break;
      }
      if (lane == 0) {
        mbar_expect_tx(&r_full[st], C::R_BYTES);
        bulk_load(r_s + st * C::R_BYTES, rec + long(ra + i) * C::R_BYTES, C::R_BYTES, &r_full[st]);
      }
    }
  } else if (warp == 8) {
    if (lane == 0) {
      constexpr uint32_t idesc = umma_idesc(128, RN, 0, 0, 0, 0);
      const uint64_t dk = umma_desc_k_sw128(smem_u32(k_s)), dq = umma_desc_k_sw128(smem_u32(r_s) + HEAD);
      bool ok = true;
      for (int i = 0; ok && i < rb - ra; ++i) {
        const int st = i % ST;
        if (!mbar_wait(&r_full[st], (i / ST) & 1, abort_flag)) { fail(ST_TIMEOUT_FULL); break; }
        const uint64_t db = dq + uint32_t(st) * (C::R_BYTES / 16);
        for (int t = 0; ok && t < n_tiles; ++t) {
          const int sb = t * 2 + (i & 1);
          ok = (i == 0 ? mbar_wait(&k_full[t], 0, abort_flag) : i < 2 || mbar_wait(&s_empty[sb], ((i >> 1) - 1) & 1, abort_flag)) ||
               fail(ST_TIMEOUT_TMEM_EMPTY);
          if (!ok) break;
          tc_fence_after();
          const uint64_t da = dk + uint32_t(t) * (C::K_BYTES / 16);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int h = 0; h < KH; ++h) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_f8(tmem + sb * RN, da + (h * 1024 + k * 2), db + ((e * KH + h) * (RN * 8) + k * 2), idesc, (e | h | k) ? 1u : 0u);
            }
          }
          umma_commit(&s_full[sb]);
        }
        if (ok) umma_commit(&r_empty[st]);
      }
    }
  } else {
    const int w = warp >> 2, tl = (warp & 3) * 32 + lane;
    const uint32_t my_lane = uint32_t((warp & 3) * 32) << 16;
    const int tok = key0 + w * BKV + tl;
    float ks = 0.f, sum = 0.f, lost = 0.f;        // the key's sum and what its additions rounded off
    if (w < n_tiles && tok < x.ctx) {
      const int blk = bt[tok / c.page];
      if (unsigned(blk) < unsigned(c.n_blocks)) ks = c.k_scale[long(blk) * c.Hkv + kvh];
      else atomicCAS(p.s.status, 0, ST_BAD_ARGS);
    }
    bool ok = true;
    for (int i = 0; i < rb - ra; ++i) {
      const int st = i % ST;
      // the record's head (its codes go to the MMA), then the scores made from it. (A warpgroup without a tile keeps step, too.)
      ok = __all_sync(0xffffffffu, mbar_wait(&r_full[st], (i / ST) & 1, abort_flag)) &&
           (w >= n_tiles || __all_sync(0xffffffffu, mbar_wait(&s_full[w * 2 + (i & 1)], (i >> 1) & 1, abort_flag)));
      if (!ok) {
        if (lane == 0) fail(ST_TIMEOUT_TMEM_FULL);
        break;
      }
      if (w < n_tiles) {
        tc_fence_after();
        const uint32_t my_S = tmem + (w * 2 + (i & 1)) * RN + my_lane;
        const float* head = reinterpret_cast<const float*>(r_s + st * C::R_BYTES);
        const int rt = ra + i, pos_a = x.base + rt * RN / G, pos_b = x.base + (min(x.rows, (rt + 1) * RN) - 1) / G;
        const int last = key0 + w * BKV + BKV - 1;
        const bool full = last < x.ctx && last <= pos_a && (p.a.window == 0 || last - BKV + 1 > pos_b - p.a.window);
        float acc0 = 0.f, acc1 = 0.f;
        auto add_up = [&](auto masked) {
#pragma unroll 2
          for (int r0 = 0; r0 < RN; r0 += 16) {
            uint32_t sr[16];
            tmem_ld16(my_S + r0, sr);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
              const float4 f4 = *reinterpret_cast<const float4*>(head + r0 + j), l4 = *reinterpret_cast<const float4*>(head + RN + r0 + j);
              const float fs[4] = {f4.x, f4.y, f4.z, f4.w}, ls[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float raw = __uint_as_float(sr[j + e]), mul = fs[e] * ks;
                float y;
                if constexpr (CAP) y = ex2(fmaf(softcap_r(raw * mul, 1.f), p.scale_log2, 0.5f * p.scale_log2) - ls[e]);
                else y = ex2(fmaf(raw, mul, -ls[e]));
                if constexpr (decltype(masked)::value) {
                  const int pos = reinterpret_cast<const int*>(head)[2 * RN + r0 + j + e];
                  if (tok > pos || tok >= x.ctx || (p.a.window > 0 && tok <= pos - p.a.window)) y = 0.f;
                }
                if (e & 1) acc1 += y;
                else acc0 += y;
              }
            }
          }
        };
        if (full) add_up(std::false_type{});        // (a branch per record, not per score)
        else add_up(std::true_type{});
        tc_fence_before();
        mbar_arrive(&s_empty[w * 2 + (i & 1)]);
        const float more = (acc0 + acc1) - lost, now = sum + more;
        lost = (now - sum) - more;
        sum = now;
      }
      if (lane == 0) mbar_arrive(&r_empty[st]);
    }
    if (ok && w < n_tiles && tok < x.ctx) p.w[seq * p.w_seq + kvh * p.w_head + tok] += sum;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 4 * RN);
  }
}

// scores [T][Hq][span] of a decode call, from the first visible tile on
__global__ void __launch_bounds__(SUM_THREADS) kv8_score_sums_kernel(const WeightArgs p, const float* scores, int span) {
  griddep_wait();
  griddep_launch();
  const int G = p.a.Hq / p.c.Hkv, kvh = blockIdx.y, seq = blockIdx.z;
  const int row = p.s.cu[seq], next = p.s.cu[seq + 1], ctx = max(p.s.ctx[seq], 0);
  if (row < 0 || row >= p.s.T || next != row + 1 || ctx > long(p.s.width) * p.c.page) return;
  const int start = (p.a.window > 0 && ctx > p.a.window) ? ctx - p.a.window : 0, base = start / BKV * BKV;
  if (ctx > p.w_keys || ctx - base > span) {
    if (threadIdx.x == 0) atomicCAS(p.s.status, 0, ST_BAD_ARGS);
    return;
  }
  const int first = base + int(blockIdx.x) * (SUM_THREADS * SUM_KEYS);
  if (first >= ctx) return;
  const int tok = first + threadIdx.x;
  const float* s = scores + (long(row) * p.a.Hq + kvh * G) * span + (tok - base);
  const float* lse = p.a.lse + long(row) * p.a.Hq + kvh * G;
  float* w = p.w + seq * p.w_seq + kvh * p.w_head + tok;
  bool in[SUM_KEYS];
  float acc[SUM_KEYS], was[SUM_KEYS];
#pragma unroll
  for (int k = 0; k < SUM_KEYS; ++k) {
    const int t = tok + k * SUM_THREADS;
    in[k] = t >= start && t < ctx;
    acc[k] = 0.f;
    was[k] = in[k] ? w[k * SUM_THREADS] : 0.f;
  }
#pragma unroll 4
  for (int g = 0; g < G; ++g) {
    const float l = lse[g], sub = l == -INFINITY ? INFINITY : l;
#pragma unroll
    for (int k = 0; k < SUM_KEYS; ++k)
      if (in[k]) acc[k] += ex2(s[long(g) * span + k * SUM_THREADS] - sub);
  }
#pragma unroll
  for (int k = 0; k < SUM_KEYS; ++k)
    if (in[k]) w[k * SUM_THREADS] = was[k] + acc[k];
}

WeightArgs make(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Attn& a, float* w, long w_seq, long w_head, int w_keys) {
  WeightArgs p{c, s, a, 0, 0, 0, 0, a.scale * 1.4426950408889634f, 0.f, w, w_seq, w_head, w_keys, nullptr};
  if (a.softcap > 0.f) {
    p.cap_k = 2.f * 1.4426950408889634f * a.scale / a.softcap;
    p.scale_log2 = 2.f * 1.4426950408889634f * a.softcap;
  }
  return p;
}

template <int KH, bool CAP>
cudaError_t launch(const CUtensorMap* tk, const WeightArgs& p, int tiles, cudaStream_t st) {
  auto kfn = kv8_weights_kernel<KH, CAP>;
  static DeviceOnce once;
  cudaError_t e = once.shared_memory(reinterpret_cast<const void*>(kfn), WCfg<KH>::SMEM);
  const dim3 records = p.packed ? dim3(unsigned(p.per_head), p.c.Hkv) : dim3(p.max_rt, p.c.Hkv, p.s.n);
  if (e == cudaSuccess) e = launch_pdl(kv8_queries_kernel<KH>, records, dim3(256), 0, st, p);
  if (e == cudaSuccess) e = launch_pdl(kfn, dim3((tiles + 1) / 2, p.c.Hkv, p.s.n), dim3(320), WCfg<KH>::SMEM, st, *tk, p);
  return e;
}

// Where the records of a call lie: by sequence, or where that has more room than its rows need (one long prompt beside 63 single tokens:
// 4.5 GB instead of 76 MB) in their order.
void place(WeightArgs& p, int observe) {
  const long G = p.a.Hq / p.c.Hkv, rows = long(observe > 0 && observe < p.s.max_new ? observe : p.s.max_new) * G;
  p.observe = observe;
  p.max_rt = int((rows + RN - 1) / RN);
  const long apart = long(p.s.n) * p.max_rt, packed = (p.s.T * G + RN - 1) / RN + p.s.n;
  p.packed = packed < apart;
  p.per_head = p.packed ? packed : apart;
}

}  // namespace

int64_t kv8_weights_scratch(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Attn& a, int observe) {
  WeightArgs p{c, s, a};
  place(p, observe);
  return int64_t(c.Hkv) * p.per_head * (HEAD + (c.dk + 127) / 128 * 2 * RN * 128);
}

int kv8_weights_launch(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Attn& a, int observe, int tiles, void* scratch, float* w, long w_seq,
                       long w_head, int w_keys, cudaStream_t st) {
  if (s.n <= 0 || s.T <= 0 || s.max_new <= 0) return 0;
  const CUtensorMap* tk = tmap_2d(c.k, uint64_t(c.n_blocks) * c.Hkv * c.page, c.dk, c.dk, c.page, 128, TM_U8, true);
  if (!tk) {
    kv8_set_error(tmap_last_error());
    return 1;
  }
  WeightArgs p = make(c, s, a, w, w_seq, w_head, w_keys);
  place(p, observe);
  p.records = static_cast<uint8_t*>(scratch);
  const bool cap = a.softcap > 0.f;
  const cudaError_t e = c.dk <= 128 ? (cap ? launch<1, true>(tk, p, tiles, st) : launch<1, false>(tk, p, tiles, st))
                                    : (cap ? launch<2, true>(tk, p, tiles, st) : launch<2, false>(tk, p, tiles, st));
  if (e != cudaSuccess) kv8_set_error(cudaGetErrorString(e));
  return e != cudaSuccess;
}

int kv8_score_sums_launch(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Attn& a, const float* scores, int span, float* w, long w_seq,
                          long w_head, int w_keys, cudaStream_t st) {
  if (s.n <= 0 || s.T <= 0) return 0;
  const WeightArgs p = make(c, s, a, w, w_seq, w_head, w_keys);
  const cudaError_t e = launch_pdl(kv8_score_sums_kernel, dim3((span + SUM_THREADS * SUM_KEYS - 1) / (SUM_THREADS * SUM_KEYS), c.Hkv, s.n),
                                   dim3(SUM_THREADS), 0, st, p, scores, span);
  if (e != cudaSuccess) kv8_set_error(cudaGetErrorString(e));
  return e != cudaSuccess;
}

}  // namespace lb
