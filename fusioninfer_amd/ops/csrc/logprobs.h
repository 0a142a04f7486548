// Launchers of logprobs.hip and of the block copies in cache.hip, as their
// bindings call them.
#pragma once

#include "common.h"

namespace fi {

constexpr int kMostChoices = 256;
constexpr int kMostBeams = 256;  // of one search
// chunks of a search's rows, of 8192 logits or more where they are many
constexpr int kMostLists = 5120;

// bytes of workspace of a call on R rows of V tokens of `size` bytes
int64_t logit_workspace(int64_t R, int V, int k, int size);

template <typename A>
void launch_beam_select(const A* logits, int64_t stride, int V,
                        const float* scores, int64_t group_stride,
                        int64_t beam_stride, int64_t G, int B, int k,
                        void* workspace, float* out_scores, int* out_parents,
                        int* out_tokens, hipStream_t stream);

template <typename A>
void launch_top_logprobs(const A* logits, int64_t stride, int64_t R, int V,
                         int k, const void* given, bool wide, void* workspace,
                         float* out_lp, int* out_ids, float* out_given,
                         hipStream_t stream);

// One tensor of blocks: `heads` pieces of `head_bytes` each, of which the first
// tokens * token_bytes are copied, a wave a slice of kSliceBytes.
struct BlockTensor {
  char* data;
  u32 head_bytes, token_bytes;
  int heads, slices;
  int blocks;
  int unit;  // bytes of one access: 16, 4 or 1
};
constexpr int kSliceBytes = 4096;
constexpr int kBlockTensors = 100;  // of one launch, its arguments hold 4 KB
struct BlockTensors {
  BlockTensor t[kBlockTensors];
};

void launch_copy_blocks(const BlockTensors& tensors, int count,
                        const int* src, const int* dst, const int* tokens,
                        int pairs, int block_size, hipStream_t stream);

}  // namespace fi
