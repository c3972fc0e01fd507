// The kernels behind the paged serving attention entries (host side).
#pragma once

#include "pb_attention_paged.cuh"

namespace pb {
namespace paged {

// CTAs that share a tree call's key tiles: so many on each SM of the current device.
uint32_t tree_ctas(uint32_t per_sm);

// Prompt attention; tree attention and the words of its workspace: binary32 elements
// on the CUDA cores.
uint32_t simt_prompt(const AttnArgs& a, uint32_t head_dim, cudaStream_t s);
uint32_t simt_tree(const AttnArgs& a, uint32_t head_dim, cudaStream_t s);
uint64_t simt_tree_words(uint32_t head_dim);

// The same on the tensor cores, for 16-bit elements; how often a wait of theirs gave up
// on the current device (added to *count, after the work of `s`).
uint32_t tc_prompt(const AttnArgs& a, uint32_t type, uint32_t head_dim, cudaStream_t s);
uint32_t tc_tree(const AttnArgs& a, uint32_t type, uint32_t head_dim, cudaStream_t s);
uint64_t tc_tree_words(uint32_t head_dim);
uint32_t tc_timeouts(cudaStream_t s, uint32_t* count);

// Tree attention of 16-bit elements with 16 * tiles rows at most on average per
// sequence and key head (tiles 1, or 2 at heads of 64).
uint32_t few_tree(const AttnArgs& a, uint32_t type, uint32_t head_dim, uint32_t tiles, cudaStream_t s);
uint64_t few_tree_words(uint32_t head_dim, uint32_t tiles);
uint32_t few_timeouts(cudaStream_t s, uint32_t* count);

// The same of binary32 elements, with row tiles of 8 or 16.
uint32_t few32_tree(const AttnArgs& a, uint32_t head_dim, uint32_t tile_rows, cudaStream_t s);
uint64_t few32_tree_words(uint32_t head_dim, uint32_t tile_rows);
uint32_t few32_timeouts(cudaStream_t s, uint32_t* count);

}  // namespace paged
}  // namespace pb
