// Moves the accepted path's rows of a paged cache to the front of the drafted region, in place, all layers in one launch.
//
// The path ascends, so row i's target (position context + i) never lies behind its source (context + path[i] >= context + i):
// going up, a row is read before another is written over it.  One thread owns one vector-wide column of a (layer, cache,
// sequence) and takes the rows in order, eight loads in flight at a time, so no two threads ever touch the same bytes and
// no barrier is needed.  Bound: the rows' bytes, read and written once; for few sequences one dependent chain
// path -> page table -> row.
#include "common.cuh"
#include "launchers.h"

namespace vkop_cuda {

constexpr int kCompactThreads = 128;

struct CompactArgs {
    unsigned char *k, *v;
    const int32_t *table, *context, *path, *count;
    int32_t *out_context;
    int64_t num_pages, table_stride;
    int64_t k_ls, k_ps, k_ts, k_hs, v_ls, v_ps, v_ts, v_hs;  // bytes
    int nodes, page_size, max_pages, columns, head_columns;  // columns: vectors in a row of all heads; of one head
    int batch, caches;
};

// Number of leading entries of the path that ascend from 0 within [0, nodes): the rows that are kept.
__device__ __forceinline__ int valid_prefix(const int32_t *path, int count, int nodes) {
    int n = min(max(count, 0), nodes);
    int ok = n;
    for (int i = threadIdx.x; i < n; i += kCompactThreads) {
        const int here = path[i], before = i > 0 ? path[i - 1] : -1;
        if (here >= nodes || here <= before)
            ok = min(ok, i);
    }
    __shared__ int s_ok;
    if (threadIdx.x == 0)
        s_ok = n;
    __syncthreads();
    if (ok < n)
        atomicMin(&s_ok, ok);
    __syncthreads();
    return s_ok;
}

template <typename V>
__global__ void __launch_bounds__(kCompactThreads) cache_compact_kernel(const CompactArgs a) {
    extern __shared__ int64_t s_row[];  // [nodes] source, [nodes] target offset of a row in its layer; -1: stays
    const int tid = threadIdx.x;
    const int layer = blockIdx.y / a.caches, which = blockIdx.y % a.caches;
    const int64_t ps = which ? a.v_ps : a.k_ps, ts = which ? a.v_ts : a.k_ts, hs = which ? a.v_hs : a.k_hs;
    unsigned char *base = which ? a.v + layer * a.v_ls : a.k + layer * a.k_ls;
    for (int b = blockIdx.z; b < a.batch; b += gridDim.z) {
        const int32_t *path = a.path + static_cast<int64_t>(b) * a.nodes;
        const int keep = valid_prefix(path, a.count[b], a.nodes);
        const int64_t context = max(a.context[b], 0);
        if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0)
            a.out_context[b] = static_cast<int32_t>(context + keep);
        for (int i = tid; i < keep; i += kCompactThreads) {
            int64_t at[2] = {context + path[i], context + i};
            bool moves = i > 0 && path[i] != i;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int64_t page = at[e] / a.page_size, slot = at[e] - page * a.page_size;
                moves = moves && page < a.max_pages;
                if (moves) {
                    const int64_t id = a.table[b * a.table_stride + page];
                    moves = id >= 0 && id < a.num_pages;
                    at[e] = id * ps + slot * ts;
                }
            }
            s_row[i] = moves ? at[0] : -1;
            s_row[a.nodes + i] = at[1];
        }
        __syncthreads();
        for (int col = blockIdx.x * kCompactThreads + tid; col < a.columns; col += gridDim.x * kCompactThreads) {
            const int head = col / a.head_columns;
            unsigned char *p = base + head * hs + static_cast<int64_t>(col - head * a.head_columns) * sizeof(V);
            for (int i0 = 1; i0 < keep; i0 += 8) {
                V r[8];
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (i0 + j < keep && s_row[i0 + j] >= 0)
                        r[j] = *reinterpret_cast<const V *>(p + s_row[i0 + j]);
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (i0 + j < keep && s_row[i0 + j] >= 0)
                        *reinterpret_cast<V *>(p + s_row[a.nodes + i0 + j]) = r[j];
            }
        }
        __syncthreads();
    }
}

int launch_cache_compact(const vkop_cache_compact_desc &d, void *k, void *v, const int32_t *table, const int32_t *context,
                         const int32_t *path, const int32_t *count, int32_t *out_context, cudaStream_t stream) {
    if (d.batch == 0)
        return VKOP_OK;
    const int64_t esz = d.dtype == VKOP_F32 ? 4 : 2;
    const int64_t dense_h = d.head_dim, dense_t = dense_h * d.kv_heads, dense_p = dense_t * d.page_size, dense_l = dense_p * d.num_pages;
    CompactArgs a;
    a.k = static_cast<unsigned char *>(k);
    a.v = static_cast<unsigned char *>(v);
    a.table = table;
    a.context = context;
    a.path = path;
    a.count = count;
    a.out_context = out_context;
    a.num_pages = d.num_pages;
    a.table_stride = d.table_stride ? d.table_stride : d.max_pages;
    a.k_ls = (d.k_layer_stride ? d.k_layer_stride : dense_l) * esz;
    a.k_ps = (d.k_page_stride ? d.k_page_stride : dense_p) * esz;
    a.k_ts = (d.k_token_stride ? d.k_token_stride : dense_t) * esz;
    a.k_hs = (d.k_head_stride ? d.k_head_stride : dense_h) * esz;
    a.v_ls = (d.v_layer_stride ? d.v_layer_stride : dense_l) * esz;
    a.v_ps = (d.v_page_stride ? d.v_page_stride : dense_p) * esz;
    a.v_ts = (d.v_token_stride ? d.v_token_stride : dense_t) * esz;
    a.v_hs = (d.v_head_stride ? d.v_head_stride : dense_h) * esz;
    a.nodes = d.nodes;
    a.page_size = d.page_size;
    a.max_pages = d.num_pages > 0 && d.layers > 0 ? d.max_pages : 0;  // without pages the table is not looked at
    a.batch = static_cast<int>(d.batch);
    a.caches = v ? 2 : 1;
    // the widest vector that every row start and head start is a multiple of
    uint64_t bits = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | static_cast<uint64_t>(d.head_dim * esz);
    for (int64_t x : {a.k_ls, a.k_ps, a.k_ts, a.k_hs})
        bits |= static_cast<uint64_t>(x);
    if (v)
        for (int64_t x : {a.v_ls, a.v_ps, a.v_ts, a.v_hs})
            bits |= static_cast<uint64_t>(x);
    const int wide = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 2;
    a.head_columns = static_cast<int>(d.head_dim * esz / wide);
    a.columns = a.head_columns * d.kv_heads;
    const dim3 grid(static_cast<unsigned>(d.layers == 0 ? 1 : (a.columns + kCompactThreads - 1) / kCompactThreads),
                    static_cast<unsigned>(d.layers == 0 ? 1 : d.layers * a.caches), static_cast<unsigned>(d.batch < 65535 ? d.batch : 65535));
    if (d.layers == 0)
        a.columns = 0;  // no rows to move; the lengths are still written
    const size_t smem = static_cast<size_t>(d.nodes) * 2 * sizeof(int64_t);
    switch (wide) {
    case 16: cache_compact_kernel<uint4><<<grid, kCompactThreads, smem, stream>>>(a); break;
    case 4: cache_compact_kernel<uint32_t><<<grid, kCompactThreads, smem, stream>>>(a); break;
    default: cache_compact_kernel<uint16_t><<<grid, kCompactThreads, smem, stream>>>(a); break;
    }
    note_launch();
    return check_launch();
}

}  // namespace vkop_cuda
