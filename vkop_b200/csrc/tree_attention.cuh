// What the kernels of the tree attention share: arguments, the tree's ancestor sets, where the parts of a row's softmax lie
// in the scratch memory, how a finished row is written.
#pragma once

#include "common.cuh"
#include "launchers.h"

namespace vkop_cuda {

constexpr int kTreeMaxNodes = 128;
constexpr int kTreeWords = kTreeMaxNodes / 32;
constexpr float kLn2 = 0.69314718055994531f;

struct TreeArgs {
    const void *q, *k, *v;
    const int32_t *table, *context, *parents, *num_nodes;
    void *out;
    float *lse;
    float *part_o;   // [batch, kv_heads, parts, rows, head_dim] unnormalised sums of a part
    float2 *part_ml; // [batch, kv_heads, parts, rows] (maximum in units of log 2, sum of exponentials)
    int64_t num_pages, table_stride;
    int64_t q_bs, q_ns, q_hs, o_bs, o_ns, o_hs;
    int64_t k_ps, k_ts, k_hs, v_ps, v_ts, v_hs;  // elements
    int64_t part_tokens;  // positions a part covers; the last part goes on to the end
    int parts;
    int batch, nodes, q_heads, kv_heads, group, head_dim, page_size, max_pages;
    int rows;             // nodes * group: the query rows that share a cache head; row r is node r / group, head r % group
    float scale_log2;     // scale * log2(e): scores are kept in units of log 2
};

__device__ __forceinline__ int tree_used(const TreeArgs &a, int b) {
    return a.num_nodes ? min(max(a.num_nodes[b], 0), a.nodes) : a.nodes;
}
__device__ __forceinline__ int64_t tree_context(const TreeArgs &a, int b) { return max(a.context[b], 0); }

// Positions to look at: those behind the table have no page.
__device__ __forceinline__ int64_t tree_length(const TreeArgs &a, int b) {
    const int64_t length = tree_context(a, b) + tree_used(a, b), width = static_cast<int64_t>(a.max_pages) * a.page_size;
    return length < width ? length : width;
}

// Parts that hold positions of a sequence of this length (one at least, which writes the empty rows too).
__device__ __forceinline__ int tree_live_parts(const TreeArgs &a, int64_t length) {
    const int64_t n = (length + a.part_tokens - 1) / a.part_tokens;
    return static_cast<int>(n < 1 ? 1 : n > a.parts ? a.parts : n);
}

// Bit j of anc[i]: node j is node i or above it.  Threads tid, tid + stride, ... fill their nodes.
__device__ __forceinline__ void tree_ancestors(const TreeArgs &a, int b, uint32_t (*anc)[kTreeWords], int tid, int stride) {
    for (int i = tid; i < a.nodes; i += stride) {
        uint32_t w[kTreeWords] = {};
        int at = i;
        while (true) {
#pragma unroll
            for (int e = 0; e < kTreeWords; e++)
                if (at >> 5 == e)
                    w[e] |= 1u << (at & 31);
            if (at == 0)
                break;
            const int up = a.parents ? a.parents[static_cast<int64_t>(b) * a.nodes + at] : at - 1;
            if (up < 0 || up >= at)  // nobody's child; and going up always ends
                break;
            at = up;
        }
#pragma unroll
        for (int e = 0; e < kTreeWords; e++)
            anc[i][e] = w[e];
    }
}

// Page of a position, or -1 where there is none.
__device__ __forceinline__ int64_t tree_page(const TreeArgs &a, int b, int64_t pos, int *slot) {
    const int64_t page = pos / a.page_size;
    *slot = static_cast<int>(pos - page * a.page_size);
    if (page >= a.max_pages)
        return -1;
    const int64_t id = a.table[b * a.table_stride + page];
    return id >= 0 && id < a.num_pages ? id : -1;
}

// launch configuration of the kernels; a plan covers every alignment of the pointers
struct TreePlan {
    int64_t part_tokens;
    int parts;
    size_t bytes;
};

// tensor-core kernel (tree_attention_mma.cu): whether type and head size suit it, its scratch, the call
bool tree_mma_serves(const vkop_tree_attention_desc &d);
size_t tree_mma_workspace(const vkop_tree_attention_desc &d);
int launch_tree_mma(const TreeArgs &args, const vkop_tree_attention_desc &d, void *workspace, cudaStream_t stream);

}  // namespace vkop_cuda
