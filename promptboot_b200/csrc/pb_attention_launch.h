// The kernels behind the paged serving attention entries (host side).
#pragma once

#include "pb_attention_paged.cuh"

namespace pb {
namespace paged {

// CTAs that share a tree call's key tiles: so many on each SM of the current device.
uint32_t tree_ctas(uint32_t per_sm);

// Prompt attention; tree attention and the words of its workspace, for rows =
// q_rows * group.
uint32_t simt_prompt(const AttnArgs& a, uint32_t type, uint32_t head_dim, cudaStream_t s);
uint32_t simt_tree(const AttnArgs& a, uint32_t type, uint32_t head_dim, cudaStream_t s);
uint64_t simt_tree_words(uint32_t head_dim, uint32_t rows, uint32_t seqs);

}  // namespace paged
}  // namespace pb
