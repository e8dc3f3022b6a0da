// Python bindings of the 8-bit key/value cache (kv8.h). Shapes and types are checked before the device, so that a refusal needs
// no GPU; what is wrong with an argument raises ValueError.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cmath>

#include "kv8.h"

namespace {
using torch::Tensor;
using OptT = c10::optional<Tensor>;

cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

#define LB_ASK(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)

lb::Kv8Cache cache_of(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs, const char* who) {
  LB_ASK(k.dim() == 4 && v.dim() == 4 && k.scalar_type() == at::kFloat8_e4m3fn && v.scalar_type() == at::kFloat8_e4m3fn &&
             k.is_contiguous() && v.is_contiguous(), who, ": codes are contiguous float8_e4m3fn [blocks, kv heads, page, head size]");
  LB_ASK(k.size(0) == v.size(0) && k.size(1) == v.size(1) && k.size(2) == v.size(2), who, ": keys and values of one cache differ in shape");
  for (const Tensor* t : {&ks, &vs})
    LB_ASK(t->dim() == 2 && t->scalar_type() == at::kFloat && t->is_contiguous() && t->size(0) == k.size(0) && t->size(1) == k.size(1), who,
           ": scales are contiguous float32 [blocks, kv heads]");
  const int64_t page = k.size(2), dk = k.size(3), dv = v.size(3);
  LB_ASK(page >= 8 && page % 8 == 0 && 64 % page == 0, who, ": pages of 8, 16, 32 or 64 tokens, not ", page);
  LB_ASK(dk >= 16 && dk <= 256 && dk % 16 == 0 && dv >= 16 && dv <= 256 && dv % 16 == 0, who,
         ": head sizes are multiples of 16 up to 256, not ", dk, " / ", dv);
  LB_ASK(k.size(0) >= 1 && k.size(1) >= 1 && (k.size(0) + 1) * k.size(1) * page < (int64_t(1) << 31), who, ": too many cells");
  LB_ASK((reinterpret_cast<uintptr_t>(k.data_ptr()) | reinterpret_cast<uintptr_t>(v.data_ptr())) % 16 == 0, who,
         ": codes start on 16 bytes");
  return {static_cast<uint8_t*>(k.data_ptr()), static_cast<uint8_t*>(v.data_ptr()), ks.data_ptr<float>(), vs.data_ptr<float>(),
          int(k.size(0)), int(k.size(1)), int(page), int(dk), int(dv)};
}

lb::Kv8Seqs seqs_of(const Tensor& table, const Tensor& ctx, const Tensor& cu, int64_t max_new, int64_t T, const Tensor& status,
                    const char* who) {
  LB_ASK(table.dim() == 2 && table.scalar_type() == at::kInt && (table.stride(1) == 1 || table.size(1) <= 1), who,
         ": the block table is int32 [sequences, blocks]");
  const int64_t n = table.size(0);
  LB_ASK(ctx.dim() == 1 && ctx.scalar_type() == at::kInt && ctx.is_contiguous() && ctx.numel() == n, who, ": lengths are int32 [sequences]");
  LB_ASK(cu.dim() == 1 && cu.scalar_type() == at::kInt && cu.is_contiguous() && cu.numel() == n + 1, who,
         ": row bounds are int32 [sequences + 1]");
  LB_ASK(n <= 65535 && T < (int64_t(1) << 31) && max_new >= 0 && max_new <= T, who, ": at most 65535 sequences, 2^31 rows, and rows of a sequence within them");
  LB_ASK(table.size(1) < (int64_t(1) << 31) / 64, who, ": table width");
  return {table.data_ptr<int>(), long(table.stride(0)), int(table.size(1)), ctx.data_ptr<int>(), cu.data_ptr<int>(), int(n), int(max_new),
          long(T), static_cast<int*>(status.data_ptr())};
}

void one_device(const Tensor& x, std::initializer_list<const Tensor*> all, const char* who) {
  for (const Tensor* t : all)
    LB_ASK(t->device() == x.device(), who, ": tensors on different devices");
  LB_ASK(x.is_cuda(), who, ": CUDA tensors");
}

// sums of weights: a row of their own for every sequence and head
void check_sums(const Tensor& w, int64_t n, int64_t heads, const char* who) {
  LB_ASK(w.dim() == 3 && w.scalar_type() == at::kFloat && w.size(0) == n && w.size(1) == heads && (w.stride(2) == 1 || w.size(2) <= 1) &&
             w.size(2) < (int64_t(1) << 31), who, ": sums of weights are float32 [sequences, kv heads, keys]");
  const int64_t L = w.size(2), a = w.stride(0), b = w.stride(1);
  const bool apart = n <= 1 ? (heads <= 1 || b >= L)
                            : heads <= 1 ? a >= L : (b >= L && a >= (heads - 1) * b + L) || (a >= L && b >= (n - 1) * a + L);
  LB_ASK(apart, who, ": rows of the sums of weights overlap");
}

void kv8_append(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs, const Tensor& new_k, const Tensor& new_v,
                const Tensor& table, const Tensor& ctx, const Tensor& cu, int64_t max_new, const Tensor& status) {
  const char* who = "kv8_append";
  const auto c = cache_of(k, v, ks, vs, who);
  for (const Tensor* t : {&new_k, &new_v})
    LB_ASK(t->dim() == 3 && t->scalar_type() == at::kBFloat16 && t->stride(2) == 1 && t->size(0) == new_k.size(0) && t->size(1) == c.Hkv, who,
           ": new keys and values are bfloat16 [rows, kv heads, head size] with neighbouring columns");
  LB_ASK(new_k.size(2) == c.dk && new_v.size(2) == c.dv, who, ": head sizes of the rows and of the cache differ");
  const auto s = seqs_of(table, ctx, cu, max_new, new_k.size(0), status, who);
  one_device(k, {&v, &ks, &vs, &new_k, &new_v, &table, &ctx, &cu, &status}, who);
  c10::cuda::CUDAGuard guard(k.device());
  const lb::Kv8Append a{new_k.data_ptr(), long(new_k.stride(0)), long(new_k.stride(1)),
                        new_v.data_ptr(), long(new_v.stride(0)), long(new_v.stride(1))};
  TORCH_CHECK(lb::kv8_append_launch(c, s, a, cur_stream()) == 0, "kv8_append: ", lb::kv8_last_error());
}

void kv8_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs, const Tensor& table,
                   const Tensor& ctx, const Tensor& cu, int64_t max_new, double scale, int64_t window, double softcap, const OptT& sink,
                   int64_t n_splits, Tensor& out, const Tensor& status, const OptT& weights, int64_t observe, int64_t tiles) {
  const char* who = "kv8_attention";
  const auto c = cache_of(k, v, ks, vs, who);
  LB_ASK(q.dim() == 3 && q.scalar_type() == at::kBFloat16 && q.stride(2) == 1 && q.size(2) == c.dk, who,
         ": queries are bfloat16 [rows, heads, head size] with neighbouring columns");
  const int64_t T = q.size(0), Hq = q.size(1);
  LB_ASK(Hq >= 1 && Hq % c.Hkv == 0 && Hq <= 65535, who, ": query heads are a multiple of the cache's heads");
  LB_ASK(window >= 0 && window < (int64_t(1) << 31) && softcap >= 0 && std::isfinite(softcap) && std::isfinite(scale), who,
         ": window and soft cap are not negative, the scale is finite");
  LB_ASK(out.scalar_type() == at::kBFloat16 && out.dim() == 3 && out.size(0) == T && out.size(1) == Hq && out.size(2) == c.dv &&
             out.stride(2) == 1 && (out.stride(1) == c.dv || Hq == 1), who, ": out is bfloat16 [rows, heads, value head size]");
  LB_ASK(T <= 1 || out.stride(0) >= Hq * c.dv, who, ": rows of out overlap");
  lb::Kv8Attn a{q.data_ptr(), long(q.stride(0)), long(q.stride(1)), int(Hq), float(scale), float(softcap), int(window), nullptr,
                out.data_ptr(), long(out.stride(0)), nullptr, nullptr, 0};
  if (sink.has_value()) {
    LB_ASK(sink->scalar_type() == at::kFloat && sink->is_contiguous() && sink->numel() == Hq && sink->device() == q.device(), who,
           ": sinks are float32 [heads]");
    a.sink = sink->data_ptr<float>();
  }
  const auto s = seqs_of(table, ctx, cu, max_new, T, status, who);
  if (weights.has_value()) {
    check_sums(*weights, s.n, c.Hkv, who);
    LB_ASK(weights->device() == q.device() && observe >= 0 && observe < (int64_t(1) << 31) && tiles >= 1 && tiles <= (int64_t(1) << 23),
           who, ": sums of weights on the queries' device, observed rows not negative");
  }
  one_device(q, {&k, &v, &ks, &vs, &table, &ctx, &cu, &out, &status}, who);
  c10::cuda::CUDAGuard guard(q.device());
  if (T == 0 || s.n == 0 || max_new == 0) return;
  LB_ASK(n_splits >= 1 && n_splits <= 255 && n_splits * c.Hkv <= 65535 && T * Hq < (int64_t(1) << 31), who, ": splits, rows");
  Tensor part;
  const int64_t nq = lb::kv8_decode_heads(int(Hq / c.Hkv)), meta = 4 * n_splits;
  if (max_new == 1) part = at::empty({meta + 2 * n_splits * nq * (c.dv + 2)}, q.options().dtype(at::kFloat));
  else if (n_splits > 1) part = at::empty({T * Hq * n_splits * (c.dv + 2)}, q.options().dtype(at::kFloat));
  Tensor lse, scratch;
  if (weights.has_value()) {
    lse = at::empty({T * Hq}, q.options().dtype(at::kFloat));
    a.lse = lse.data_ptr<float>();
    if (max_new == 1) {
      scratch = at::empty({T * Hq * tiles * 128}, q.options().dtype(at::kFloat));
      a.scores = scratch.data_ptr<float>();
      a.span = int(tiles * 128);
    } else {
      scratch = at::empty({lb::kv8_weights_scratch(c, s, a, int(observe))}, q.options().dtype(at::kByte));
    }
  }
  float* pp = part.defined() ? part.data_ptr<float>() : nullptr;
  const int rc = max_new == 1 ? lb::kv8_decode_launch(c, s, a, int(n_splits), pp + meta, reinterpret_cast<int*>(pp), cur_stream())
                              : lb::kv8_prompt_launch(c, s, a, int(n_splits), pp, cur_stream());
  TORCH_CHECK(rc == 0, "kv8_attention: ", lb::kv8_last_error());
  if (!weights.has_value()) return;
  float* w = weights->data_ptr<float>();
  const long ws = long(weights->stride(0)), wh = long(weights->stride(1));
  const int keys = int(weights->size(2));
  const int wc = max_new == 1 ? lb::kv8_score_sums_launch(c, s, a, a.scores, a.span, w, ws, wh, keys, cur_stream())
                              : lb::kv8_weights_launch(c, s, a, int(observe), int(tiles), scratch.data_ptr(), w, ws, wh, keys, cur_stream());
  TORCH_CHECK(wc == 0, "kv8_attention: ", lb::kv8_last_error());
}

void kv8_evict(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs, const Tensor& table, const Tensor& ctx,
               const Tensor& weights, int64_t budget, int64_t first, int64_t last, const Tensor& dst, Tensor& lens, Tensor& kept,
               Tensor& w_out, const Tensor& status) {
  const char* who = "kv8_evict";
  const auto c = cache_of(k, v, ks, vs, who);
  LB_ASK(table.dim() == 2 && table.scalar_type() == at::kInt && (table.stride(1) == 1 || table.size(1) <= 1) && dst.dim() == 2 &&
             dst.scalar_type() == at::kInt && (dst.stride(1) == 1 || dst.size(1) <= 1) && dst.size(0) == table.size(0), who,
         ": block tables are int32 [sequences, blocks]");
  const int64_t n = table.size(0);
  LB_ASK(ctx.dim() == 1 && ctx.scalar_type() == at::kInt && ctx.is_contiguous() && ctx.numel() == n, who, ": lengths are int32 [sequences]");
  LB_ASK(n <= 65535 && table.size(1) < (int64_t(1) << 31) / 64, who, ": at most 65535 sequences");
  LB_ASK(budget >= 1 && budget < (int64_t(1) << 30) && first >= 0 && last >= 0 && first + last <= budget, who,
         ": the budget holds the first and last tokens that stay");
  LB_ASK(dst.size(1) * c.page >= budget, who, ": the blocks of the result hold fewer tokens than the budget");
  check_sums(weights, n, c.Hkv, who);
  for (const Tensor* t : {&kept, &w_out})
    LB_ASK(t->dim() == 3 && t->is_contiguous() && t->size(0) == n && t->size(1) == c.Hkv && t->size(2) == budget, who, ": results");
  LB_ASK(lens.scalar_type() == at::kInt && kept.scalar_type() == at::kInt && w_out.scalar_type() == at::kFloat && lens.numel() == n &&
             lens.is_contiguous(), who, ": results");
  one_device(k, {&v, &ks, &vs, &table, &ctx, &weights, &dst, &lens, &kept, &w_out, &status}, who);
  c10::cuda::CUDAGuard guard(k.device());
  const lb::Kv8Seqs s{table.data_ptr<int>(), long(table.stride(0)), int(table.size(1)), ctx.data_ptr<int>(), nullptr, int(n), 0, 0,
                      static_cast<int*>(status.data_ptr())};
  const lb::Kv8Evict e{weights.data_ptr<float>(), long(weights.stride(0)), long(weights.stride(1)), int(weights.size(2)), int(budget),
                       int(first), int(last), dst.data_ptr<int>(), long(dst.stride(0)), lens.data_ptr<int>(), kept.data_ptr<int>(),
                       w_out.data_ptr<float>()};
  TORCH_CHECK(lb::kv8_evict_launch(c, s, e, cur_stream()) == 0, "kv8_evict: ", lb::kv8_last_error());
}
}  // namespace

void bind_kv8(pybind11::module_& m) {
  m.def("kv8_append", &kv8_append);
  m.def("kv8_attention", &kv8_attention);
  m.def("kv8_evict", &kv8_evict);
}
