// PyTorch bindings of the operators that a search with beams runs on:
// log-probabilities and the choice of beams (logprobs.hip), copies of cache
// blocks and state slots (cache.hip). Every entry checks its operands against
// what kernel and grid assume, and runs on the device of its operands, on the
// current stream there.

#include <torch/extension.h>

#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>

#include <tuple>
#include <vector>

#include "logprobs.h"

namespace {

using fi::u16;
using Guard = c10::hip::OptionalHIPGuardMasqueradingAsCUDA;

hipStream_t current_stream() {
  return c10::hip::getCurrentHIPStream().stream();
}

void check_launch() {
  const hipError_t e = hipGetLastError();
  TORCH_CHECK(e == hipSuccess, "launch failed: ", hipGetErrorString(e));
}

// Checks raise ValueError, as those of CPU operands do.
#define CHECK_THAT(ok, ...) TORCH_CHECK_VALUE(ok, __VA_ARGS__)

// rows with their tokens one after another
at::Tensor rows_of(const at::Tensor& t) {
  CHECK_THAT(t.is_cuda() && t.dim() == 2 && t.size(1) >= 1,
             "logits are rows of at least one token");
  CHECK_THAT(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16,
             "logits are float32 or bfloat16");
  // a grid holds 2^32 threads, at most one workgroup for 1024 logits or row
  CHECK_THAT(t.size(1) < (1ll << 30) &&
                 t.size(0) * (t.size(1) / 1024 + 1) < (1ll << 24),
             "too many logits in one call");
  if (t.stride(1) == 1 || t.size(1) == 1) return t;
  return t.contiguous();
}

void check_search(int64_t beams, int64_t tokens) {
  CHECK_THAT(beams * ((tokens + 8191) / 8192) <= fi::kMostLists, beams,
             " beams over ", tokens, " tokens are too many in one search");
}

// scores [G, k], parents [G, k], tokens [G, k]
std::tuple<at::Tensor, at::Tensor, at::Tensor> beam_select(
    const at::Tensor& of, const at::Tensor& scores, int64_t k) {
  const at::Tensor logits = rows_of(of);
  CHECK_THAT(k >= 1 && k <= fi::kMostChoices, "k is ", k, ", not from 1 to ",
             fi::kMostChoices);
  CHECK_THAT(scores.dim() == 2 && scores.scalar_type() == at::kFloat &&
                 scores.device() == logits.device(),
             "scores are float32 [searches, beams] on the device of the "
             "logits");
  const int64_t G = scores.size(0), B = scores.size(1);
  CHECK_THAT(G * B == logits.size(0) && B >= 1 && B <= fi::kMostBeams,
             logits.size(0), " rows of logits for [", G, ", ", B, "] beams");
  check_search(B, logits.size(1));
  const Guard guard(logits.device());
  const auto f32 = logits.options().dtype(at::kFloat);
  const auto i32 = logits.options().dtype(at::kInt);
  at::Tensor s = at::empty({G, k}, f32);
  at::Tensor p = at::empty({G, k}, i32), t = at::empty({G, k}, i32);
  if (G == 0) return {s, p, t};
  const int V = logits.size(1);
  at::Tensor ws = at::empty({fi::logit_workspace(G * B, V, std::min<int64_t>(k, V),
                                                 logits.element_size())},
                            logits.options().dtype(at::kByte));
  const auto run = [&](auto* x) {
    fi::launch_beam_select(x, logits.stride(0), V, scores.data_ptr<float>(),
                           scores.stride(0), scores.stride(1), G, B, k,
                           ws.data_ptr(), s.data_ptr<float>(),
                           p.data_ptr<int>(), t.data_ptr<int>(),
                           current_stream());
  };
  if (logits.scalar_type() == at::kFloat)
    run(logits.data_ptr<float>());
  else
    run(static_cast<const u16*>(logits.data_ptr()));
  check_launch();
  return {s, p, t};
}

// log-probabilities [R, k], tokens [R, k], of the given tokens [R]
std::tuple<at::Tensor, at::Tensor, c10::optional<at::Tensor>> top_logprobs(
    const at::Tensor& from, int64_t k,
    const c10::optional<at::Tensor>& token_ids) {
  const at::Tensor logits = rows_of(from);
  const int64_t R = logits.size(0);
  const int64_t most = std::min<int64_t>(fi::kMostChoices, logits.size(1));
  CHECK_THAT(k >= 0 && k <= most, "k is ", k, ", not from 0 to ", most);
  check_search(1, logits.size(1));
  c10::optional<at::Tensor> given;
  if (token_ids) {
    CHECK_THAT(token_ids->device() == logits.device() &&
                   token_ids->dim() == 1 && token_ids->size(0) == R &&
                   (token_ids->scalar_type() == at::kInt ||
                    token_ids->scalar_type() == at::kLong),
               "token_ids are int32 or int64, one for each row, on its "
               "device");
    given = token_ids->contiguous();
  }
  const Guard guard(logits.device());
  const auto f32 = logits.options().dtype(at::kFloat);
  at::Tensor lp = at::empty({R, k}, f32);
  at::Tensor ids = at::empty({R, k}, logits.options().dtype(at::kInt));
  c10::optional<at::Tensor> of;
  if (given) of = at::empty({R}, f32);
  if (R == 0 || (k == 0 && !given)) return {lp, ids, of};
  const int V = logits.size(1);
  at::Tensor ws = at::empty({fi::logit_workspace(R, V, k, logits.element_size())},
                            logits.options().dtype(at::kByte));
  const bool wide = given && given->scalar_type() == at::kLong;
  const auto run = [&](auto* x) {
    fi::launch_top_logprobs(x, logits.stride(0), R, V, k,
                            given ? given->data_ptr() : nullptr, wide,
                            ws.data_ptr(), lp.data_ptr<float>(),
                            ids.data_ptr<int>(),
                            of ? of->data_ptr<float>() : nullptr,
                            current_stream());
  };
  if (logits.scalar_type() == at::kFloat)
    run(logits.data_ptr<float>());
  else
    run(static_cast<const u16*>(logits.data_ptr()));
  check_launch();
  return {lp, ids, of};
}

void copy_blocks(const std::vector<at::Tensor>& tensors,
                 const at::Tensor& src_ids, const at::Tensor& dst_ids,
                 const c10::optional<at::Tensor>& token_counts) {
  const int64_t pairs = src_ids.numel();
  const auto ids = [&](const at::Tensor& t) {
    CHECK_THAT(t.scalar_type() == at::kInt,
               "src, dst and tokens are int32");
    CHECK_THAT(t.dim() == 1 && t.numel() == pairs,
               "src, dst and tokens hold one value for each pair");
    CHECK_THAT(t.is_cuda() && t.device() == src_ids.device(),
               "tensors and ids are on one device");
    return t.contiguous();
  };
  const at::Tensor src = ids(src_ids), dst = ids(dst_ids);
  c10::optional<at::Tensor> tokens;
  if (token_counts) tokens = ids(*token_counts);
  CHECK_THAT(pairs < (1ll << 31), "too many pairs");
  // every tensor is checked before the first launch
  std::vector<fi::BlockTensors> tables;
  int64_t count = 0;
  int block_size = -1;
  for (const auto& t : tensors) {
    CHECK_THAT(t.dim() >= 1 && t.is_contiguous(),
               "tensors of blocks are contiguous");
    CHECK_THAT(t.device() == src.device(),
               "tensors and ids are on one device");
    if (tokens) {
      CHECK_THAT(t.dim() == 4 && t.size(2) < (1ll << 31) &&
                     (block_size < 0 || t.size(2) == block_size),
                 "tokens go with paged tensors [blocks, heads, block_size, "
                 "width] of one block_size");
      block_size = static_cast<int>(t.size(2));
    }
    if (pairs == 0 || t.numel() == 0) continue;
    const int64_t block = t.numel() / t.size(0) * t.element_size();
    const int64_t heads = tokens ? t.size(1) : 1;
    const int64_t token = tokens ? t.size(3) * t.element_size() : block;
    CHECK_THAT(block < (1ll << 31) && t.size(0) < (1ll << 31),
               "a block must be smaller than 2 GiB");
    const auto bits =
        reinterpret_cast<uintptr_t>(t.data_ptr()) | block | token;
    const int64_t at = count++ % fi::kBlockTensors;
    if (at == 0) tables.emplace_back();
    fi::BlockTensor& e = tables.back().t[at];
    e.data = static_cast<char*>(t.data_ptr());
    e.head_bytes = static_cast<fi::u32>(block / heads);
    e.token_bytes = static_cast<fi::u32>(token);
    e.heads = static_cast<int>(heads);
    e.slices = static_cast<int>((block / heads + fi::kSliceBytes - 1) /
                                fi::kSliceBytes);
    e.blocks = static_cast<int>(t.size(0));
    e.unit = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
  }
  const Guard guard(src.device());
  for (const auto& table : tables) {
    fi::launch_copy_blocks(table, std::min<int64_t>(count, fi::kBlockTensors),
                           src.data_ptr<int>(), dst.data_ptr<int>(),
                           tokens ? tokens->data_ptr<int>() : nullptr, pairs,
                           block_size, current_stream());
    check_launch();
    count -= fi::kBlockTensors;
  }
}

}  // namespace

void register_search_ops(pybind11::module& m) {
  m.def("beam_select", &beam_select, "the k best continuations of every search");
  m.def("top_logprobs", &top_logprobs, "top and given log-probabilities");
  m.def("copy_blocks", &copy_blocks, "blocks of tensors onto others");
}
