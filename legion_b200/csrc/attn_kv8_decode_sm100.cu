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
// the denominator adds exp(z) 2^-e (in 32 bits: a weight of 2^-37 next to a value scale 2^100 times its own).
//
// One CTA per SM, and all of them share the batch's tiles evenly: the tiles of all (sequence, kv head) groups in a row, cut into
// equal stretches, whatever the lengths are. A stretch ends one group, has some whole ones and begins another; a CTA goes through
// its pieces without draining: loads and scores run ahead into the next piece. A whole group's result is written at once, parts
// of a group go to scratch for kv8_combine_kernel. (A CTA per group and split paid 7 us for its first tile and its end each time:
// 64 sequences of 750 to 2250 tokens, 40 / 8 heads of 128, took 94 us.) Scratch belongs to the call.
//
// Two softmax warpgroups (warps 0..3 and 4..7; thread = key of the tile, later output column) take alternate tiles, each a
// stream of its own with its P and O^T; they meet in shared memory at the end of a piece. Warp 8: the scores' MMAs, four tiles ahead
// of their softmax (a wait for a phase of a stage's barrier cannot miss it: the stage's next scores stand behind P of this tile,
// the stage's next P V behind P of the tile that waits). Warps 9, 12: TMA of keys and of values through the block table into as
// many stages as fit (six of 32 KB for heads of 128), and the tiles' scales. Warp 10: the next piece's queries. Warp 11: P V. Code
// that runs once a piece or rarely is kept short: unrolled over the heads it was fetched at 6000 clocks a piece.
//
// 16 sequences of 8192 tokens, 32 / 4 heads of 128: 37.4 us = 3.6 TB/s with the join, 0.55 of the measured copy rate. In its steady
// state a tile takes an SM 1200 to 1370 clocks, which is the memory's rate; the rest is the launch's beginning (lengths, table,
// first keys: dependent reads, and instructions fetched behind them) and its end.
#include "kv8_dev.cuh"
#include "tmap.cuh"

namespace lb {
namespace {

struct DecodeArgs {
  Kv8Cache c;
  Kv8Seqs s;
  Kv8Attn a;
  int cells;                    // of a row of the table
  float scale_log2, cap_k;      // as in softcap_r: soft-capped scores have 2 cap log2(e) in scale_log2
  float* part;                  // [CTAs][2][NQ][dv + 2]: sums over the values, reference (log2), denominator; 0: the piece that a
                                // CTA begins with, 1: the one it ends with, where they are parts of a group
  int4* meta;                   // [CTAs]: row, first head, heads, parts of the group that begins in this CTA's last piece (0: none)
};

// P is taken relative to the reference times 2^11, and the reference moves when a weight passes it by more than 2^4: at most 2^15,
// which e5m2 and a half hold, and e5m2's last step, 2^-16, lies 2^-27 below the largest weight. (A reference within 2^2 moved in a
// quarter of the tiles of a stream of 2000 keys, 1900 clocks each.)
constexpr float OFFSET = 11.f;
constexpr float SLACK = 4.f;

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
  static constexpr int Q_BYTES = KH * NS * 128, P_BYTES = NO * 128;
  static constexpr int SEQS = 128;                                         // lengths kept in shared memory
  static constexpr int SC = 1472, SEQ = SC + 16 * 16 * 8;       // offsets in the tail
  static constexpr int TAIL = SEQ + SEQS * 8;
  // P of a tile may be written while P V two tiles back still reads the other buffer, where four stages or more are left (with
  // three, the wait for P V four tiles back could miss its phase)
  static constexpr int ROOM = 227 * 1024 - TAIL - 1024 - 2 * Q_BYTES;
  static constexpr int TWO = (ROOM - 4 * P_BYTES) / (K_BYTES + V_BYTES), ONE = (ROOM - 2 * P_BYTES) / (K_BYTES + V_BYTES);
  static constexpr int PB = TWO >= 4 ? 2 : 1;                              // P buffers of a warpgroup
  static constexpr int STAGES = PB == 2 ? (TWO > 6 ? 6 : TWO) : (ONE > 6 ? 6 : ONE);
  static constexpr int SMEM = STAGES * (K_BYTES + V_BYTES) + 2 * Q_BYTES + 2 * PB * P_BYTES + TAIL + 1024;
  static constexpr int LA = STAGES < 4 ? STAGES : 4;                       // tiles whose scores are made ahead
  static constexpr int TMEM_RAW = LA * NS + 2 * MT * NO;
  static constexpr int TMEM_COLS = TMEM_RAW <= 128 ? 128 : TMEM_RAW <= 256 ? 256 : 512;
  static_assert(TMEM_RAW <= 512 && STAGES >= 3 && STAGES <= 6 && SMEM <= 227 * 1024 && (PB == 1 || STAGES >= 4) && P_BYTES >= 8 * 128 * 4, "sizes");
};

// A sequence's first tile, tiles (at least one if it has a row: a row that sees nothing is a result, too), length and row
struct SeqInfo {
  int tile0, tiles, ctx, row;
};
__device__ __forceinline__ SeqInfo seq_info(int ctx, int row, int window) {
  SeqInfo r;
  const int start = (window > 0 && ctx > window) ? ctx - window : 0;
  r.tile0 = start / 128;
  r.tiles = row < 0 ? 0 : max(1, (ctx + 127) / 128 - r.tile0);
  r.ctx = ctx;
  r.row = row;
  return r;
}

// The pieces of a CTA: (sequence, head group, tiles t .. t + n of it), walked by every role for itself
template <typename F>
struct Pieces {
  const F& seq;                   // index -> SeqInfo
  int groups, n_seqs;
  int b, hg, t, left;
  SeqInfo i;
  __device__ Pieces(const F& f, int groups_, int n_seqs_, int b_, int hg_, int t_, int left_)
      : seq(f), groups(groups_), n_seqs(n_seqs_), b(b_), hg(hg_), t(t_), left(left_), i(f(b_)) {}
  __device__ int n() const { return min(i.tiles - t, left); }
  __device__ void next() {
    left -= n();
    t = 0;
    if (left > 0 && ++hg == groups) {
      hg = 0;
      do {
        ++b;
        i = seq(b);
      } while (i.tiles == 0 && b + 1 < n_seqs);
    }
  }
};

// SCORES: they are left in a.scores
template <int KH, int MT, int NQ, bool CAP, bool SCORES>
__global__ void __launch_bounds__(416, 1)
kv8_decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const DecodeArgs p) {
  using C = Cfg<KH, MT, NQ>;
  constexpr int BKV = C::BKV, NS = C::NS, NO = C::NO, ST = C::STAGES, LA = C::LA, PB = C::PB;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* k_s = smem;
  uint8_t* v_s = k_s + ST * C::K_BYTES;
  uint8_t* q_s = v_s + ST * C::V_BYTES;                   // [2]
  uint8_t* p_s = q_s + 2 * C::Q_BYTES;                    // [2 warpgroups][PB], each on 1024 bytes
  uint8_t* tail = p_s + 2 * PB * C::P_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(tail);
  uint64_t* k_full = bars;         // [6] one per stage
  uint64_t* k_done = bars + 6;     // scores made: for the softmax, and the stage is free
  uint64_t* v_full = bars + 12;
  uint64_t* v_done = bars + 18;    // P V done: P may be written, O touched, and the stage is free
  uint64_t* p_ready = bars + 24;   // [4] tile % 4: a warpgroup may be through with a tile before P V of its last one is issued
  uint64_t* q_free = bars + 28;    // [2] scores of a piece made
  uint64_t* q_full = bars + 30;    // [8] a piece's queries and their power of two
  uint64_t* sc_full = bars + 38;   // [16] a tile's scales
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 54);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* s_red = reinterpret_cast<float*>(tail + 512);    // [2 warpgroups][NQ][4 warps] maxima, then sums
  float* s_ref = reinterpret_cast<float*>(tail + 1024);   // [2 warpgroups][references NQ, factors NQ]
  float2* s_fac = reinterpret_cast<float2*>(tail + 1280); // [NQ] what each warpgroup's sums count in the result
  float* fq_s = reinterpret_cast<float*>(tail + 1408);    // [8]
  int* s_start = reinterpret_cast<int*>(tail + 1440);     // sequence, group, tile, units, and the batch's units (64 bits)
  float* s_sc = reinterpret_cast<float*>(tail + C::SC);   // [16][keys, values][16] a tile's scales per 8 keys
  int2* s_seq = reinterpret_cast<int2*>(tail + C::SEQ);   // length, row (-1: none)

  const Kv8Cache& c = p.c;
  const int G = p.a.Hq / c.Hkv, gtiles = (G + NQ - 1) / NQ, groups = c.Hkv * gtiles, n_seqs = p.s.n;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 1) {                 // (one thread for all barriers took a microsecond)
    if (lane < 24) mbar_init(bars + lane, 1);                            // stages
    else if (lane < 28) mbar_init(bars + lane, 128);                     // p_ready
    else if (lane < 30) mbar_init(bars + lane, 1);                       // q_free
    if (lane < 8) mbar_init(&q_full[lane], 32);
    else if (lane < 24) mbar_init(&sc_full[lane - 8], 64);
    if (lane == 0) *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  griddep_wait();
  griddep_launch();
  auto read_seq = [&](int b) -> int2 {
    const int row = p.s.cu[b], end = p.s.cu[b + 1];
    const int ctx = max(p.s.ctx[b], 0);
    const bool good = row >= 0 && end <= p.s.T && end <= row + 1 && (end <= row || ctx <= p.cells);
    if (!good && blockIdx.x == 0) atomicCAS(p.s.status, 0, ST_BAD_ARGS);
    return make_int2(ctx, good && end == row + 1 ? row : -1);
  };
  if (warp == 0) {
    // every lane adds up a stretch of the sequences; the lane whose stretch holds this CTA's first tile finds it
    const int per = (n_seqs + 31) / 32, lo = min(n_seqs, lane * per), hi = min(n_seqs, lo + per);
    long mine = 0;
    for (int b = lo; b < hi; ++b) {
      const int2 x = read_seq(b);
      if (b < C::SEQS) s_seq[b] = x;
      mine += seq_info(x.x, x.y, p.a.window).tiles;
    }
    long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    const long total = __shfl_sync(0xffffffffu, inc, 31) * groups;
    const long n_cta = min(long(gridDim.x), total);           // those with work: each has a tile at least
    const bool mine_too = blockIdx.x < n_cta;
    const long u0 = mine_too ? total * blockIdx.x / n_cta : 0, u1 = mine_too ? total * (blockIdx.x + 1) / n_cta : 0;
    if (lane == 0) {
      s_start[3] = int(u1 - u0);
      *reinterpret_cast<long*>(s_start + 4) = total;
    }
    const long from = (inc - mine) * groups;
    if (u1 > u0 && u0 >= from && u0 < inc * groups) {
      long at = u0 - from;
      for (int b = lo; b < hi; ++b) {
        const int2 x = read_seq(b);
        const int t = seq_info(x.x, x.y, p.a.window).tiles;
        if (at < long(t) * groups) {
          s_start[0] = b;
          s_start[1] = int(at / t);
          s_start[2] = int(at % t);
          break;
        }
        at -= long(t) * groups;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t tmem_S = tmem_base, tmem_O = tmem_base + LA * NS;
  const int ppb = BKV / c.page;
  const int D = c.dv;
  const int units = s_start[3];
  const long total = *reinterpret_cast<long*>(s_start + 4);
  const auto seq = [&](int b) {
    const int2 x = b < C::SEQS ? s_seq[b] : read_seq(b);
    return seq_info(x.x, x.y, p.a.window);
  };
  if (units <= 0 && threadIdx.x == 0) p.meta[blockIdx.x] = make_int4(0, 0, 0, 0);

  if (units <= 0) {
  } else if (warp == 9 || warp == 12) {
    // ------------------------------------------------------------------ TMA, keys (warp 9) and values (warp 12): the lanes hold
    // the rows of the next 32 pages and their scales, lane 0 issues. Table entries and scales are fetched a fill ahead, into the
    // next piece too. (One warp for both issued a tile in 2000 clocks.)
    const bool val = warp == 12;
    const CUtensorMap* tm = val ? &tmV : &tmK;
    uint64_t* full = val ? v_full : k_full;
    uint64_t* done = val ? v_done : k_done;
    const float* scales = val ? c.v_scale : c.k_scale;
    const int parts = val ? MT : KH, bytes = val ? C::V_BYTES : C::K_BYTES;
    uint8_t* ring = val ? v_s : k_s;
    const int fill = 32 / ppb;                             // tiles
    using P = Pieces<decltype(seq)>;
    P s(seq, groups, n_seqs, s_start[0], s_start[1], s_start[2], units);
    // (block, head) of this lane's page of the tiles from j on; -1 behind the sequence
    auto unit_of = [&](const P& x, int j) -> long {
      const long page = long(x.i.tile0 + x.t + j) * ppb + lane;
      if (page * c.page >= x.i.ctx || j * ppb + lane >= x.n() * ppb) return -1;
      const int blk = p.s.table[x.b * p.s.ld_table + page];
      if (unsigned(blk) >= unsigned(c.n_blocks)) {
        atomicCAS(p.s.status, 0, ST_BAD_ARGS);
        return -1;
      }
      return long(blk) * c.Hkv + x.hg / gtiles;
    };
    long next = unit_of(s, 0);
    float next_sc = next >= 0 ? scales[next] : 0.f;
    bool ok = true;
    int it = 0, st = 0, lap = 0;
    for (; ok && s.left > 0; s.next()) {
      const int n = s.n();
      int row = 0;
      float sc = 0.f;
      for (int j = 0; ok && j < n; ++j, ++it) {
        const int slot = j % fill;
        if (slot == 0) {
          // a page behind the sequence, or a block outside the cache: rows that TMA fills with zeros
          row = int(next >= 0 ? next : long(c.n_blocks) * c.Hkv) * c.page;
          sc = val ? kv8_value_scale(next_sc) : next_sc;
          if (j + fill < n) {
            next = unit_of(s, j + fill);
          } else if (s.left > n) {
            P x = s;
            x.next();
            next = unit_of(x, 0);
          }
        }
        if (it >= ST && !__all_sync(0xffffffffu, mbar_wait(&done[st], (lap - 1) & 1, abort_flag))) {
          if (lane == 0) { *abort_flag = 1; atomicCAS(p.s.status, 0, ST_TIMEOUT_EMPTY | SITE_DECODE_ATTN); }
          ok = false;
          break;
        }
        uint8_t* dst = ring + st * bytes;
        if (lane == 0) mbar_expect_tx(&full[st], bytes);
        for (int g = 0; g < ppb; ++g) {
          const int r = __shfl_sync(0xffffffffu, row, slot * ppb + g);
          if (lane == 0) {
            tma_load_2d(dst + g * c.page * 128, tm, &full[st], 0, r);
            if (parts == 2) tma_load_2d(dst + BKV * 128 + g * c.page * 128, tm, &full[st], 128, r);
          }
        }
        // slot it % 16 held tile it - 16, whose softmax is over: this stage is free, so scores (and P V) ST tiles back are made, and
        // scores stand behind P of the tile LA <= 4 before
        const float a = __shfl_sync(0xffffffffu, sc, slot * ppb + (lane & 15) * 8 / c.page);
        if (lane < 16) s_sc[((it & 15) * 2 + (val ? 1 : 0)) * 16 + lane] = a;
        mbar_arrive(&sc_full[it & 15]);
        if (slot == 1 || j + 1 == n || fill == 1) next_sc = next >= 0 ? scales[next] : 0.f;
        if (++st == ST) {
          st = 0;
          ++lap;
        }
      }
    }
  } else if (warp == 8) {
    // ------------------------------------------------------------------ scores (one thread issues)
    // Descriptors are made once; a step adds its offset in 16-byte units. (Made anew for every MMA they take the issuing thread
    // 170 clocks each; an MMA of this shape takes 40.)
    if (lane == 0) {
      constexpr uint32_t idesc = umma_idesc(128, NS, 0, 0, 0, 0);         // e4m3 x e4m3
      const uint64_t dk = umma_desc_k_sw128(smem_u32(k_s)), dq = umma_desc_k_sw128(smem_u32(q_s));
      bool ok = true;
      int i = 0, sn = 0;
      for (Pieces<decltype(seq)> s(seq, groups, n_seqs, s_start[0], s_start[1], s_start[2], units); ok && s.left > 0; s.next(), ++sn) {
        const int end = i + s.n();
        ok = mbar_wait(&q_full[sn & 7], (sn >> 3) & 1, abort_flag);
        const uint64_t db = dq + uint32_t(sn & 1) * (C::Q_BYTES / 16);
        for (; ok && i < end; ++i) {
          const int st = i % ST;
          // into the buffer of tile i - LA, which its softmax has read
          ok = (i < LA || mbar_wait(&p_ready[(i - LA) & 3], ((i - LA) >> 2) & 1, abort_flag)) && mbar_wait(&k_full[st], (i / ST) & 1, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint64_t da = dk + uint32_t(st) * (C::K_BYTES / 16);
          const uint32_t ts = tmem_S + (i % LA) * NS;
#pragma unroll
          for (int h = 0; h < KH; ++h) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_f8(ts, da + (h * (BKV * 8) + k * 2), db + (h * (NS * 8) + k * 2), idesc, (h | k) ? 1u : 0u);
          }
          umma_commit(&k_done[st]);
        }
        if (ok) umma_commit(&q_free[sn & 1]);
      }
      if (!ok) { *abort_flag = 1; atomicCAS(p.s.status, 0, ST_TIMEOUT_FULL | SITE_DECODE_ATTN); }
    }
  } else if (warp == 11) {
    // ------------------------------------------------------------------ P V (one thread issues; beside the scores' thread: one
    // thread for both took 1100 clocks a tile, four fifths of what its bytes take)
    if (lane == 0) {
      constexpr uint32_t idesc = umma_idesc(128, NO, 0, 1, 1, 0);         // e4m3 (V^T, MN-major) x e5m2
      const uint64_t dv = umma_desc_mn_sw128(smem_u32(v_s), BKV * 128, 1024), dp = umma_desc_k_sw128(smem_u32(p_s));
      bool ok = true;
      int i = 0;
      for (Pieces<decltype(seq)> s(seq, groups, n_seqs, s_start[0], s_start[1], s_start[2], units); ok && s.left > 0; s.next()) {
        const int begin = i, end = i + s.n();
        for (; ok && i < end; ++i) {
          const int st = i % ST;
          ok = mbar_wait(&p_ready[i & 3], (i >> 2) & 1, abort_flag) && mbar_wait(&v_full[st], (i / ST) & 1, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint64_t da = dv + uint32_t(st) * (C::V_BYTES / 16), db = dp + uint32_t((i & 1) * PB + (i >> 1) % PB) * (C::P_BYTES / 16);
          const uint32_t to = tmem_O + (i & 1) * MT * NO, more = i - begin >= 2;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int k = 0; k < BKV / 32; ++k)
              umma_f8(to + mt * NO, da + (mt * (BKV * 8) + k * 256), db + k * 2, idesc, k ? 1u : more);
          }
          umma_commit(&v_done[st]);
        }
      }
      if (!ok) { *abort_flag = 1; atomicCAS(p.s.status, 0, ST_TIMEOUT_FLAG | SITE_DECODE_ATTN); }
    }
  } else if (warp == 10) {
    // ------------------------------------------------------------------ queries of the pieces
    // One power of two for all heads of a piece (what a smaller head loses is 2^-21 of the largest query value, and a softmax sees
    // absolute errors of its scores); a value that is not finite is a NaN code and makes its head NaN.
    constexpr int PER = NQ * KH / 4;                                    // chunks of 16 values of a lane
    int sn = 0;
    bool ok = true;
    for (Pieces<decltype(seq)> s(seq, groups, n_seqs, s_start[0], s_start[1], s_start[2], units); s.left > 0; s.next(), ++sn) {
      const int kvh = s.hg / gtiles, g0 = (s.hg % gtiles) * NQ, gn = min(NQ, G - g0);
      uint32_t u[PER][8];
      uint32_t m = 0;
#pragma unroll
      for (int r = 0; r < PER; ++r) {
        const int q = (lane + r * 32) / (KH * 8), ch = (lane + r * 32) % (KH * 8);
#pragma unroll
        for (int i = 0; i < 8; ++i) u[r][i] = 0u;
        if (q < gn && ch * 16 < c.dk) {
          const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(p.a.q) + s.i.row * p.a.q_tok + (kvh * G + g0 + q) * p.a.q_head + ch * 16;
          if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
            *reinterpret_cast<uint4*>(u[r]) = reinterpret_cast<const uint4*>(src)[0];
            *reinterpret_cast<uint4*>(u[r] + 4) = reinterpret_cast<const uint4*>(src)[1];
          } else {
            const uint16_t* hsrc = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
            for (int i = 0; i < 8; ++i) u[r][i] = hsrc[2 * i] | uint32_t(hsrc[2 * i + 1]) << 16;
          }
        }
      }
#pragma unroll
      for (int r = 0; r < PER; ++r) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t lo = u[r][i] & 0x7fffu, hi = (u[r][i] >> 16) & 0x7fffu;
          m = max(m, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
        }
      }
      m = __reduce_max_sync(0xffffffffu, m);
      const float qs = kv8_scale_of(__uint_as_float(m << 16)), inv = kv8_inverse(qs);
      // the buffer held the queries of two pieces ago
      if (ok && sn >= 2 && !__all_sync(0xffffffffu, mbar_wait(&q_free[sn & 1], ((sn >> 1) - 1) & 1, abort_flag))) {
        *abort_flag = 1;
        atomicCAS(p.s.status, 0, ST_TIMEOUT_EMPTY | SITE_DECODE_ATTN);
        ok = false;
      }
      uint8_t* qb = q_s + (sn & 1) * C::Q_BYTES;
#pragma unroll
      for (int r = 0; r < PER; ++r) {
        const int q = (lane + r * 32) / (KH * 8), ch = (lane + r * 32) % (KH * 8);
        uint32_t hi4[4], lo4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          hi4[i] = lo4[i] = 0u;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t x = u[r][2 * i + j];
            const float a0 = __uint_as_float(x << 16) * inv, a1 = __uint_as_float(x & 0xffff0000u) * inv;
            uint32_t hh = e4m3x2(a0, a1);
            if ((x & 0x7f80u) == 0x7f80u) hh |= 0x7fu;
            if ((x & 0x7f800000u) == 0x7f800000u) hh |= 0x7f00u;
            const float2 f = __half22float2(e4m3x2_to_half2(hh));
            hi4[i] |= hh << (16 * j);
            lo4[i] |= e4m3x2((a0 - f.x) * 16.f, (a1 - f.y) * 16.f) << (16 * j);
          }
        }
        if (ok) {
          const uint32_t at = (ch / 8) * (NS * 128) + q * 128 + (((ch & 7) ^ (q & 7)) << 4);
          *reinterpret_cast<uint4*>(qb + at) = make_uint4(hi4[0], hi4[1], hi4[2], hi4[3]);
          *reinterpret_cast<uint4*>(qb + at + NQ * 128) = make_uint4(lo4[0], lo4[1], lo4[2], lo4[3]);
        }
      }
      // (eight slots: scores run at most four tiles, so four pieces ahead, queries two more)
      if (lane == 0) fq_s[sn & 7] = qs * (CAP ? p.cap_k : p.scale_log2);
      fence_proxy_async_smem();
      mbar_arrive(&q_full[sn & 7]);
    }
  } else {
    // ------------------------------------------------------------------ softmax (warps 0..7)
    const int w = warp >> 2, wq = warp & 3, tl = wq * 32 + lane;
    const uint32_t lane_off = uint32_t(wq * 32) << 16;
    const uint32_t my_S = tmem_S + lane_off, my_O = tmem_O + w * MT * NO + lane_off;
    const int bar_id = 1 + w;
    float* red = s_red + w * (NQ * 4);
    float* s_m = s_ref + w * (2 * NQ);                           // references of the heads, and what O shrank by last
    float* s_alpha = s_m + NQ;
    float* x_s = reinterpret_cast<float*>(p_s + PB * C::P_BYTES);      // the second warpgroup's P, idle at the end of a piece
    // A wait that runs out does not leave the loops: the warp keeps taking part in the named barriers, without waiting again.
    bool ok = true;
    auto fail = [&](int code) { *abort_flag = 1; atomicCAS(p.s.status, 0, code | SITE_DECODE_ATTN); ok = false; };
    int it = 0, sn = 0;
    for (Pieces<decltype(seq)> s(seq, groups, n_seqs, s_start[0], s_start[1], s_start[2], units); s.left > 0; s.next(), ++sn) {
      const int g0 = (s.hg % gtiles) * NQ, gn = min(NQ, G - g0), head0 = (s.hg / gtiles) * G + g0;
      const int n = s.n(), tile0 = s.i.tile0 + s.t, ctx = s.i.ctx, row = s.i.row;
      const int start = (p.a.window > 0 && ctx > p.a.window) ? ctx - p.a.window : 0;
      if (ok && !__all_sync(0xffffffffu, mbar_wait(&q_full[sn & 7], (sn >> 3) & 1, abort_flag))) fail(ST_TIMEOUT_FULL);
      const float fq = fq_s[sn & 7];
      float m_ref[NQ], l_run[NQ];
#pragma unroll
      for (int q = 0; q < NQ; ++q) { m_ref[q] = -INFINITY; l_run[q] = 0.f; }
      if (tl < NQ) s_m[tl] = -INFINITY;        // (nobody reads the last piece's any more)
      int n_mine = 0;
      const int end = it + n;
      for (int i = it + ((it ^ w) & 1); i < end; i += 2, ++n_mine) {
        if (ok && !__all_sync(0xffffffffu, mbar_wait(&sc_full[i & 15], (i >> 4) & 1, abort_flag))) fail(ST_TIMEOUT_FULL);
        const float mul = fq * s_sc[(i & 15) * 32 + (tl >> 3)];
        const int ev = kv8_log2(s_sc[(i & 15) * 32 + 16 + (tl >> 3)]);
        const float add = float(ev), inv_v = __uint_as_float(uint32_t(127 - ev) << 23);     // |ev| <= 120
        if (ok && !__all_sync(0xffffffffu, mbar_wait(&k_done[i % ST], (i / ST) & 1, abort_flag))) fail(ST_TIMEOUT_TMEM_FULL);
        uint32_t r[NS];
#pragma unroll
        for (int q = 0; q < NS; ++q) r[q] = 0u;
        if (ok) {
          tc_fence_after();
          tm_ld<NS>(my_S + (i % LA) * NS, r);
          tmem_ld_wait();
        }
        const int key0 = (tile0 + i - it) * BKV, tok = key0 + tl;
        const bool valid = tok >= start && tok < ctx;
        float* sc_out = nullptr;
        if constexpr (SCORES) {
          const int rel = tok - s.i.tile0 * BKV;
          if (valid && rel < p.a.span) sc_out = p.a.scores + (long(row) * p.a.Hq + head0) * p.a.span + rel;
        }
        float z[NQ];
        bool over = false;
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          z[q] = -INFINITY;
          if (q < gn) {
            float x = fmaf(__uint_as_float(r[NQ + q]), 0.0625f, __uint_as_float(r[q])) * mul;
            if constexpr (CAP) x = fmaf(softcap_r(x, 1.f), p.scale_log2, 0.5f * p.scale_log2);
            if (SCORES && sc_out) sc_out[q * long(p.a.span)] = x;
            if (valid) z[q] = x + add;
            over |= z[q] > m_ref[q] + SLACK;
          }
        }
        uint32_t any_over;
        asm volatile(
            "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, %2, 128, p;\n\t"
            "selp.u32 %0, 1, 0, q;\n\t}"
            : "=r"(any_over) : "r"(over ? 1u : 0u), "r"(bar_id) : "memory");
        // the P V that read this P buffer; where O moves, the one before
        const int back = any_over || PB == 1 ? 2 : 4;
        if (ok && n_mine >= back / 2 && !__all_sync(0xffffffffu, mbar_wait(&v_done[(i - back) % ST], ((i - back) / ST) & 1, abort_flag)))
          fail(ST_TIMEOUT_TMEM_EMPTY);
        uint8_t* my_p = p_s + (w * PB + (i >> 1) % PB) * C::P_BYTES;
        if (any_over) {
          // a thread per head finds its new reference, and what sums and O shrink by; everybody takes them from shared memory
#pragma unroll
          for (int q = 0; q < NQ; ++q) {
            float wm;
            asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(wm) : "f"(z[q]));
            if (lane == q) red[q * 4 + wq] = wm;
          }
          asm volatile("bar.sync %0, 128;" ::"r"(bar_id) : "memory");
          if (tl < NQ) {
            const float4 m4 = *reinterpret_cast<const float4*>(&red[tl * 4]);
            const float old = s_m[tl], m = fmaxf(fmaxf(fmaxf(m4.x, m4.y), fmaxf(m4.z, m4.w)), old);
            s_alpha[tl] = old == -INFINITY ? 0.f : ex2(old - m);
            s_m[tl] = m;
          }
          asm volatile("bar.sync %0, 128;" ::"r"(bar_id) : "memory");
          float alpha[NQ];
#pragma unroll
          for (int q = 0; q < NQ; q += 4) {
            *reinterpret_cast<float4*>(alpha + q) = *reinterpret_cast<const float4*>(s_alpha + q);
            *reinterpret_cast<float4*>(m_ref + q) = *reinterpret_cast<const float4*>(s_m + q);
          }
#pragma unroll
          for (int q = 0; q < NQ; ++q) l_run[q] *= alpha[q];
          if (ok && n_mine >= 1) {
            tc_fence_after();
#pragma unroll 1
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
        }
        // P: [term * NQ + head][key], K-major rows of 128 bytes, 128-byte swizzle. (Rows of heads that do not exist are columns of O
        // that nobody reads.)
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
        mbar_arrive(&p_ready[i & 3]);
      }
      it = end;
      if (ok && n_mine >= 1) {
        const int last = end - 1 - ((end - 1 - w) & 1);
        if (!__all_sync(0xffffffffu, mbar_wait(&v_done[last % ST], (last / ST) & 1, abort_flag))) fail(ST_TIMEOUT_TMEM_FULL);
      }
      // ---- end of a piece: sums over the keys, the second warpgroup hands its results to the first, eight heads at a time
      const bool whole = s.t == 0 && n == s.i.tiles;
      float* part = p.part + ((long(blockIdx.x) * 2 + (s.t == 0 ? 1 : 0)) * NQ) * (D + 2);
      // (lanes trade halves of the heads until each holds one head's sum over its lanes)
#pragma unroll
      for (int o = NQ / 2; o >= 1; o >>= 1) {
        const bool up = lane & o;
#pragma unroll
        for (int q = 0; q < o; ++q) {
          const float keep = up ? l_run[q + o] : l_run[q], give = up ? l_run[q] : l_run[q + o];
          l_run[q] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
      }
#pragma unroll
      for (int o = NQ; o < 32; o <<= 1) l_run[0] += __shfl_xor_sync(0xffffffffu, l_run[0], o);
      if (lane < NQ) red[lane * 4 + wq] = l_run[0];
      named_sync<3, 256>();
      if (threadIdx.x < NQ) {
        const int q = threadIdx.x;
        const float4 a4 = *reinterpret_cast<const float4*>(&s_red[q * 4]), b4 = *reinterpret_cast<const float4*>(&s_red[(NQ + q) * 4]);
        const float l0 = (a4.x + a4.y) + (a4.z + a4.w), l1 = (b4.x + b4.y) + (b4.z + b4.w);
        const float m0 = s_ref[q], m1 = s_ref[2 * NQ + q], m = fmaxf(m0, m1);
        float f0 = m0 == -INFINITY ? (l0 == l0 ? 0.f : 1.f) : ex2(m0 - m);      // (NaN passes)
        float f1 = m1 == -INFINITY ? (l1 == l1 ? 0.f : 1.f) : ex2(m1 - m);
        float den = l0 * f0 + l1 * f1, top = m == -INFINITY ? m : m - OFFSET;
        if (q < gn && whole) {
          float f = 1.f;
          if (p.a.sink) f = kv8_add_sink(p.a.sink[head0 + q] * 1.4426950408889634f, top, den);
          const float inv = den > 0.f || den != den ? f / den : 0.f;
          f0 *= inv;
          f1 *= inv;
          if (p.a.lse) p.a.lse[long(row) * p.a.Hq + head0 + q] = den > 0.f ? top + log2f(den) : -INFINITY;
        } else if (q < gn) {
          part[q * (D + 2) + D] = top;
          part[q * (D + 2) + D + 1] = den;
        }
        s_fac[q] = make_float2(f0, f1);
      }
      tc_fence_after();
#pragma unroll 1
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll 1
        for (int h0 = 0; h0 < gn; h0 += 8) {
          uint32_t o[3][8];
#pragma unroll
          for (int t = 0; t < 3; ++t) {
#pragma unroll
            for (int j = 0; j < 8; ++j) o[t][j] = 0u;
          }
          if (ok && n_mine >= 1) {
#pragma unroll
            for (int t = 0; t < 3; ++t)
              asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                           : "=r"(o[t][0]), "=r"(o[t][1]), "=r"(o[t][2]), "=r"(o[t][3]), "=r"(o[t][4]), "=r"(o[t][5]), "=r"(o[t][6]),
                             "=r"(o[t][7])
                           : "r"(my_O + mt * NO + t * NQ + h0) : "memory");
            tmem_ld_wait();
          }
          if (w == 1) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              x_s[j * 128 + tl] = __uint_as_float(o[0][j]) + (__uint_as_float(o[1][j]) + __uint_as_float(o[2][j]));
          }
          named_sync<3, 256>();
          const int d = mt * 128 + tl;
          if (w == 0 && d < D && !*abort_flag) {
            __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.a.out) + row * p.a.o_tok + (head0 + h0) * D + d;
            float* pd = part + h0 * (D + 2) + d;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float2 f = s_fac[h0 + j];
              const float v = (__uint_as_float(o[0][j]) + (__uint_as_float(o[1][j]) + __uint_as_float(o[2][j]))) * f.x + x_s[j * 128 + tl] * f.y;
              if (h0 + j < gn) {
                if (whole) dst[j * D] = __float2bfloat16(v);
                else pd[j * (D + 2)] = v;
              }
            }
          }
          named_sync<3, 256>();
        }
      }
      if (threadIdx.x == 0 && s.left == n) {
        // the last piece: if a group begins here and goes on, how many CTAs hold its parts
        int parts = 0;
        if (s.t == 0 && !whole) {
          const long n_cta = min(long(gridDim.x), total), last = total * (blockIdx.x + 1) / n_cta + (s.i.tiles - n) - 1;
          parts = int(((last + 1) * n_cta - 1) / total) - int(blockIdx.x) + 1;
        }
        p.meta[blockIdx.x] = make_int4(row, head0, gn, parts);
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

// Joins partial results: sum over parts of 2^(m - M) O, over the sum of 2^(m - M) l (and a sink). `at(i)`: part i, dv + 2 floats.
template <typename F>
__device__ __forceinline__ void join(const Kv8Attn& a, int D, long row, int h, int parts, F at, float* s_w) {
  const float sk = a.sink ? a.sink[h] * 1.4426950408889634f : -INFINITY;
  if (threadIdx.x < 32) {
    float m = sk;
    for (int i = threadIdx.x; i < parts; i += 32) m = fmaxf(m, at(i)[D]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float l = 0.f;
    for (int i = threadIdx.x; i < parts; i += 32) {
      const float mi = at(i)[D], li = at(i)[D + 1];
      const float f = mi == -INFINITY ? (li == li ? 0.f : 1.f) : ex2(mi - m);
      l += f * li;
      s_w[i] = f;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (sk != -INFINITY) l += ex2(sk - m);
    if (threadIdx.x == 0) {
      s_w[255] = l > 0.f || l != l ? 1.f / l : 0.f;
      if (a.lse) a.lse[row * a.Hq + h] = l > 0.f ? m + log2f(l) : -INFINITY;
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += 128) {
    float o = 0.f;
#pragma unroll 8
    for (int i = 0; i < parts; ++i) o += s_w[i] * at(i)[d];
    static_cast<__nv_bfloat16*>(a.out)[row * a.o_tok + h * D + d] = __float2bfloat16(o * s_w[255]);
  }
}

// Groups of the decode kernel that lie in several CTAs: a CTA here for each of them and each head of a group
__global__ void __launch_bounds__(128) kv8_combine_kernel(const DecodeArgs p, int nq) {
  __shared__ float s_w[256];
  griddep_wait();
  griddep_launch();
  const int4 m = p.meta[blockIdx.x];
  const int q = blockIdx.y;
  if (m.w == 0 || q >= m.z) return;
  const long stride = long(p.c.dv + 2);
  join(p.a, p.c.dv, m.x, m.y + q, m.w,
       [&](int i) { return p.part + ((long(blockIdx.x + i) * 2 + (i == 0 ? 1 : 0)) * nq + q) * stride; }, s_w);
}

// Prompt rows: every part of every row and head is there, but for rows of no sequence and of those that the attention leaves out
__global__ void __launch_bounds__(128) kv8_join_kernel(const Kv8Seqs s, const Kv8Attn a, int page, int D, int n_splits, const float* part) {
  __shared__ float s_w[256];
  const int h = blockIdx.x % a.Hq;
  const long row = blockIdx.x / a.Hq;
  int seq = 0;                                             // the last sequence that begins here or before
  for (int end = s.n; end - seq > 1;) {
    const int mid = (seq + end) / 2;
    if (s.cu[mid] <= row) seq = mid;
    else end = mid;
  }
  const int q0 = s.cu[seq], q1 = s.cu[seq + 1];
  if (q0 < 0 || row < q0 || row >= q1 || q1 > s.T || q1 - q0 > s.max_new || s.ctx[seq] > long(s.width) * page) return;
  join(a, D, row, h, n_splits, [&](int i) { return part + ((row * a.Hq + h) * n_splits + i) * (D + 2); }, s_w);
}

template <int KH, int MT, int NQ, bool CAP, bool SCORES>
cudaError_t launch(const CUtensorMap* tk, const CUtensorMap* tv, const DecodeArgs& p, int ctas, cudaStream_t st) {
  auto kfn = kv8_decode_kernel<KH, MT, NQ, CAP, SCORES>;
  constexpr int smem = Cfg<KH, MT, NQ>::SMEM;
  static DeviceOnce once;
  const cudaError_t e = once.shared_memory(reinterpret_cast<const void*>(kfn), smem);
  if (e != cudaSuccess) return e;
  return launch_pdl(kfn, dim3(ctas), dim3(416), smem, st, *tk, *tv, p);
}

}  // namespace

cudaError_t kv8_join(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Attn& a, int n_splits, float* part, cudaStream_t st) {
  kv8_join_kernel<<<unsigned(s.T * a.Hq), 128, 0, st>>>(s, a, c.page, c.dv, n_splits, part);
  return cudaGetLastError();
}

int kv8_decode_heads(int group) { return group <= 8 ? 8 : 16; }

int kv8_decode_launch(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Attn& a, int ctas, float* part, int* meta, cudaStream_t st) {
  if (s.n <= 0 || s.T <= 0) return 0;
  const uint64_t rows = uint64_t(c.n_blocks) * c.Hkv * c.page;
  const CUtensorMap* tk = tmap_2d(c.k, rows, c.dk, c.dk, c.page, 128, TM_U8, true);
  const CUtensorMap* tv = tmap_2d(c.v, rows, c.dv, c.dv, c.page, 128, TM_U8, true);
  if (!tk || !tv) {
    kv8_set_error(tmap_last_error());
    return 1;
  }
  DecodeArgs p{c, s, a, s.width * c.page, a.scale * 1.4426950408889634f, 0.f, part, reinterpret_cast<int4*>(meta)};
  const bool cap = a.softcap > 0.f;
  if (cap) {
    p.cap_k = 2.f * 1.4426950408889634f * a.scale / a.softcap;
    p.scale_log2 = 2.f * 1.4426950408889634f * a.softcap;
  }
  const int kh = (c.dk + 127) / 128, mt = (c.dv + 127) / 128, nq = kv8_decode_heads(a.Hq / c.Hkv);
  cudaError_t e = cudaErrorInvalidValue;
#define LB_KV8(K_, V_, Q_)                                                                                                      \
  if (kh == K_ && mt == V_ && nq == Q_)                                                                                         \
    e = a.scores ? (cap ? launch<K_, V_, Q_, true, true>(tk, tv, p, ctas, st) : launch<K_, V_, Q_, false, true>(tk, tv, p, ctas, st)) \
                 : (cap ? launch<K_, V_, Q_, true, false>(tk, tv, p, ctas, st) : launch<K_, V_, Q_, false, false>(tk, tv, p, ctas, st));
  LB_KV8(1, 1, 8) LB_KV8(1, 1, 16) LB_KV8(2, 2, 8) LB_KV8(2, 2, 16) LB_KV8(1, 2, 8) LB_KV8(1, 2, 16) LB_KV8(2, 1, 8) LB_KV8(2, 1, 16)
#undef LB_KV8
  if (e == cudaSuccess && ctas > 1) e = launch_pdl(kv8_combine_kernel, dim3(ctas, nq), dim3(128), 0, st, p, nq);
  if (e != cudaSuccess) kv8_set_error(cudaGetErrorString(e));
  return e != cudaSuccess;
}

}  // namespace lb
