// Launch interface of the 8-bit key/value cache (kv8_cache.cu, kv8_evict.cu, attn_kv8_decode_sm100.cu,
// attn_kv8_prompt_sm100.cu, kv8_weights_sm100.cu). A cache is e4m3 codes
// [blocks, kv heads, page, head size] for keys and for values and one float32 scale, a power of two, per block and head
// [blocks, kv heads]; a value is its code times its block's scale. Pointers are device pointers; every function returns 0 on
// success and enqueues without synchronising.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace lb {

struct Kv8Cache {
  uint8_t* k; uint8_t* v;
  float* k_scale; float* v_scale;
  int n_blocks, Hkv, page, dk, dv;
};

// Sequences of a call: sequence i owns query (or new) rows cu[i] .. cu[i + 1], the last of its ctx[i] tokens, which lie in the
// blocks of row i of the table. A length beyond the table: kv8_append leaves out the rows behind it, attention the sequence, which it
// records (ST_BAD_ARGS).
struct Kv8Seqs {
  const int* table; long ld_table; int width;
  const int* ctx; const int* cu;
  int n, max_new;
  long T;                          // rows of the call
  int* status;
};

struct Kv8Append {
  const void* k; long k_tok, k_head;    // bf16 [T, kv heads, dk]: elements between tokens and between heads
  const void* v; long v_tok, v_head;
};
int kv8_append_launch(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Append& a, cudaStream_t st);

struct Kv8Attn {
  const void* q; long q_tok, q_head;    // bf16 [T, Hq, dk]
  int Hq;
  float scale, softcap;
  int window;
  const float* sink;                    // [Hq] or nullptr
  void* out; long o_tok;                // bf16 [T, Hq * dv], elements between rows
  float* lse;                           // [T, Hq] log2 of the sum of the exponentials, or nullptr
  float* scores; int span;              // decode: [T, Hq, span] takes the scores (log2) from the first visible tile on, or nullptr
};
// Decode (max_new == 1) on `ctas` CTAs, 255 at most. part: 2 * ctas * kv8_decode_heads(Hq / Hkv) * (dv + 2) floats, meta: 4 * ctas ints
// on 16 bytes.
int kv8_decode_launch(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Attn& a, int ctas, float* part, int* meta, cudaStream_t st);
int kv8_decode_heads(int group);
// Prompts and rows behind a context: the tiles of 128 keys that a tile of rows sees fall into n_splits parts.
// part: n_splits * (dv + 2) floats for every row and head, where n_splits > 1.
int kv8_prompt_launch(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Attn& a, int n_splits, float* part, cudaStream_t st);
// Joins the partial results of every row and head of a prompt call.
cudaError_t kv8_join(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Attn& a, int n_splits, float* part, cudaStream_t st);
// w[sequence, kv head, key] += softmax weights of the sequence's last `observe` rows (0: all), with a.lse from the attention. Rows of
// prompts: the longest context has `tiles` tiles of 128 keys at most; scratch of kv8_weights_scratch bytes, on 16 bytes. Decode: from
// the scores that the attention left in a.scores.
int kv8_weights_launch(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Attn& a, int observe, int tiles, void* scratch, float* w, long w_seq,
                       long w_head, int w_keys, cudaStream_t st);
int64_t kv8_weights_scratch(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Attn& a, int observe);
int kv8_score_sums_launch(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Attn& a, const float* scores, int span, float* w, long w_seq,
                          long w_head, int w_keys, cudaStream_t st);

// Eviction: of every sequence and kv head the first `first` tokens, the last `last` and those of the largest weights stay, `budget`
// in all, in order, in the blocks of dst. s.cu and s.max_new are not used.
struct Kv8Evict {
  const float* w; long w_seq, w_head; int w_keys;
  int budget, first, last;
  const int* dst; long ld_dst;
  int* lens;                            // [sequences]
  int* kept;                            // [sequences, kv heads, budget], -1 behind the last
  float* w_out;                         // likewise, 0 behind the last
};
int kv8_evict_launch(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Evict& e, cudaStream_t st);
const char* kv8_last_error();
void kv8_set_error(const char* what);

}  // namespace lb
