// Attention of a tree of drafted tokens over a paged cache: the general kernel, the join of a row's parts, and the choice
// between the kernels.
//
// The positions of a sequence are cut into parts that different CTAs take; each part leaves the maximum m, the sum l of
// exp2(s - m) and the sum of exp2(s - m) v of every row, and the join adds the parts up with weights exp2(m - max m), in
// the order of the parts.  A sequence that is one part long is written out at once.
#include "tree_attention.cuh"

namespace vkop_cuda {

// ---- general kernel: any of the three types, any head size that is a multiple of 8, any strides ----
//
// One warp a query row, eight rows a CTA; the CTA's rows share tiles of 32 keys and values in shared memory (32 bits).  A
// lane takes one key's score, then a column of the values.  It serves 32-bit tensors and layouts that the tensor-core
// kernel cannot take; its arithmetic (2 x 2 x rows x positions x head_dim FMAs from shared memory) bounds it.
constexpr int kGenWarps = 8;
constexpr int kGenTile = 32;
constexpr int kGenMaxDim = 256;

template <typename T>
__global__ void __launch_bounds__(kGenWarps * 32) tree_attention_general_kernel(const TreeArgs a) {
    extern __shared__ float s_f[];
    const int D = a.head_dim, pad = D + 1;
    float *s_k = s_f, *s_v = s_k + kGenTile * pad, *s_q = s_v + kGenTile * pad;
    __shared__ uint32_t s_anc[kTreeMaxNodes][kTreeWords];
    __shared__ int64_t s_page[kGenTile];
    __shared__ int s_slot[kGenTile];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int part = blockIdx.x, b = blockIdx.z;
    const int h = blockIdx.y % a.kv_heads, r = blockIdx.y / a.kv_heads * kGenWarps + warp;
    const int used = tree_used(a, b);
    const int64_t context = tree_context(a, b), length = tree_length(a, b);
    const int live = tree_live_parts(a, length);
    if (part >= live)
        return;
    const int64_t begin = part * a.part_tokens, end = part == a.parts - 1 ? length : min(length, begin + a.part_tokens);
    const bool row_ok = r < a.rows;
    const int node = row_ok ? r / a.group : 0, head = h * a.group + (row_ok ? r % a.group : 0);
    const bool row_live = row_ok && node < used;
    tree_ancestors(a, b, s_anc, tid, kGenWarps * 32);
    if (row_ok)
        for (int d = lane; d < D; d += 32)
            s_q[warp * D + d] = Elem<T>::from_storage(static_cast<const T *>(a.q)[b * a.q_bs + node * a.q_ns + head * a.q_hs + d]);
    float m = -INFINITY, l = 0.0f, acc[kGenMaxDim / 32];
#pragma unroll
    for (int e = 0; e < kGenMaxDim / 32; e++)
        acc[e] = 0.0f;
    for (int64_t t0 = begin; t0 < end; t0 += kGenTile) {
        __syncthreads();
        if (tid < kGenTile) {
            int slot = 0;
            s_page[tid] = t0 + tid < end ? tree_page(a, b, t0 + tid, &slot) : -1;
            s_slot[tid] = slot;
        }
        __syncthreads();
        for (int i = tid; i < kGenTile * D; i += kGenWarps * 32) {
            const int t = i / D, d = i - t * D;
            const int64_t page = s_page[t];
            float kv = 0.0f, vv = 0.0f;
            if (page >= 0) {
                kv = Elem<T>::from_storage(static_cast<const T *>(a.k)[page * a.k_ps + s_slot[t] * a.k_ts + h * a.k_hs + d]);
                vv = Elem<T>::from_storage(static_cast<const T *>(a.v)[page * a.v_ps + s_slot[t] * a.v_ts + h * a.v_hs + d]);
            }
            s_k[t * pad + d] = kv;
            s_v[t * pad + d] = vv;
        }
        __syncthreads();
        if (!row_live)
            continue;
        const int64_t pos = t0 + lane;
        bool sees = s_page[lane] >= 0;
        if (sees && pos >= context) {
            const int j = static_cast<int>(pos - context);
            sees = s_anc[node][j >> 5] >> (j & 31) & 1u;
        }
        float dot = 0.0f;
        for (int d = 0; d < D; d++)
            dot = fmaf(s_q[warp * D + d], s_k[lane * pad + d], dot);
        const float s = sees ? dot * a.scale_log2 : -INFINITY;
        const float top = fmaxf(m, warp_max(s)), base = top == -INFINITY ? 0.0f : top;
        const float keep = exp2f(m - base), p = sees ? exp2f(s - base) : 0.0f;
        l = l * keep + warp_sum(p);
        m = top;
#pragma unroll
        for (int e = 0; e < kGenMaxDim / 32; e++)
            acc[e] *= keep;
        for (unsigned left = __ballot_sync(kFullMask, sees); left; left &= left - 1) {
            const int t = __ffs(left) - 1;
            const float w = __shfl_sync(kFullMask, p, t);
#pragma unroll
            for (int e = 0; e < kGenMaxDim / 32; e++)
                if (lane + 32 * e < D)
                    acc[e] = fmaf(w, s_v[t * pad + lane + 32 * e], acc[e]);
        }
    }
    if (!row_ok)
        return;
    if (live == 1) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        T *o = static_cast<T *>(a.out) + b * a.o_bs + node * a.o_ns + head * a.o_hs;
#pragma unroll
        for (int e = 0; e < kGenMaxDim / 32; e++)
            if (lane + 32 * e < D)
                o[lane + 32 * e] = Elem<T>::to_storage(l == 0.0f ? 0.0f : acc[e] * inv);
        if (a.lse && lane == 0)
            a.lse[(static_cast<int64_t>(b) * a.nodes + node) * a.q_heads + head] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
    } else {
        const int64_t at = ((static_cast<int64_t>(b) * a.kv_heads + h) * a.parts + part) * a.rows + r;
#pragma unroll
        for (int e = 0; e < kGenMaxDim / 32; e++)
            if (lane + 32 * e < D)
                a.part_o[at * D + lane + 32 * e] = acc[e];
        if (lane == 0)
            a.part_ml[at] = make_float2(m, l);
    }
}

// ---- join: one warp a row ----
constexpr int kJoinWarps = 4;

template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32) tree_attention_join_kernel(const TreeArgs a) {
    const int lane = threadIdx.x & 31, D = a.head_dim;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kJoinWarps + (threadIdx.x >> 5);  // (b * kv_heads + h) * rows + r
    if (row >= static_cast<int64_t>(a.batch) * a.kv_heads * a.rows)
        return;
    const int64_t unit = row / a.rows;
    const int r = static_cast<int>(row - unit * a.rows), b = static_cast<int>(unit / a.kv_heads), h = static_cast<int>(unit % a.kv_heads);
    const int live = tree_live_parts(a, tree_length(a, b));
    if (live == 1)
        return;
    const int64_t at = unit * a.parts * a.rows + r;
    float top = -INFINITY;
    for (int p = lane; p < live; p += 32)
        top = fmaxf(top, a.part_ml[at + static_cast<int64_t>(p) * a.rows].x);
    top = warp_max(top);
    const float base = top == -INFINITY ? 0.0f : top;
    float l = 0.0f, acc[kGenMaxDim / 32];
#pragma unroll
    for (int e = 0; e < kGenMaxDim / 32; e++)
        acc[e] = 0.0f;
    for (int p = 0; p < live; p++) {
        const int64_t i = at + static_cast<int64_t>(p) * a.rows;
        const float2 ml = a.part_ml[i];
        const float w = exp2f(ml.x - base);
        l = fmaf(w, ml.y, l);
#pragma unroll
        for (int e = 0; e < kGenMaxDim / 32; e++)
            if (lane + 32 * e < D)
                acc[e] = fmaf(w, a.part_o[i * D + lane + 32 * e], acc[e]);
    }
    const int node = r / a.group, head = h * a.group + r % a.group;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T *o = static_cast<T *>(a.out) + b * a.o_bs + node * a.o_ns + head * a.o_hs;
#pragma unroll
    for (int e = 0; e < kGenMaxDim / 32; e++)
        if (lane + 32 * e < D)
            o[lane + 32 * e] = Elem<T>::to_storage(l == 0.0f ? 0.0f : acc[e] * inv);
    if (a.lse && lane == 0)
        a.lse[(static_cast<int64_t>(b) * a.nodes + node) * a.q_heads + head] = l == 0.0f ? -INFINITY : (top + log2f(l)) * kLn2;
}

// Parts for a kernel that takes `rows_a_cta` rows with one CTA: about `ctas` CTAs in all, none shorter than `least` positions.
static TreePlan plan_parts(const vkop_tree_attention_desc &d, int rows_a_cta, int64_t ctas, int64_t least) {
    const int64_t rows = static_cast<int64_t>(d.nodes) * (d.q_heads / d.kv_heads);
    const int64_t units = d.batch * d.kv_heads * ((rows + rows_a_cta - 1) / rows_a_cta);
    int64_t longest = d.max_context > 0 ? d.max_context : static_cast<int64_t>(d.max_pages) * d.page_size;
    longest += d.nodes;
    int64_t parts = units > 0 ? (ctas + units - 1) / units : 1;
    const int64_t most = (longest + least - 1) / least;
    parts = parts > most ? most : parts;
    parts = parts < 1 ? 1 : parts > 4096 ? 4096 : parts;
    TreePlan p;
    p.part_tokens = ((longest + parts - 1) / parts + 127) / 128 * 128;
    p.parts = static_cast<int>((longest + p.part_tokens - 1) / p.part_tokens);
    p.bytes = p.parts == 1 ? 0 : static_cast<size_t>(d.batch) * d.kv_heads * p.parts * rows * (d.head_dim + 2) * sizeof(float);
    return p;
}

static TreePlan plan_general(const vkop_tree_attention_desc &d) { return plan_parts(d, kGenWarps, 148 * 4, 512); }

int plan_tree_attention(const vkop_tree_attention_desc &d, size_t *bytes) {
    *bytes = plan_general(d).bytes;
    if (tree_mma_serves(d)) {  // the pointers' alignment decides at the call
        const size_t mma = tree_mma_workspace(d);
        *bytes = *bytes > mma ? *bytes : mma;
    }
    return VKOP_OK;
}

template <typename T>
static int launch_general(const TreeArgs &a, const TreePlan &plan, cudaStream_t stream) {
    const size_t smem = static_cast<size_t>(2 * kGenTile * (a.head_dim + 1) + kGenWarps * a.head_dim) * sizeof(float);
    if (smem > 32 * 1024 && cudaFuncSetAttribute(tree_attention_general_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 static_cast<int>(smem)) != cudaSuccess) {
        cudaGetLastError();
        return VKOP_CUDA_ERROR;
    }
    const dim3 grid(static_cast<unsigned>(plan.parts), static_cast<unsigned>((a.rows + kGenWarps - 1) / kGenWarps * a.kv_heads),
                    static_cast<unsigned>(a.batch));
    tree_attention_general_kernel<T><<<grid, kGenWarps * 32, smem, stream>>>(a);
    note_launch();
    return check_launch();
}

template <typename T>
static int launch_t(TreeArgs &a, const vkop_tree_attention_desc &d, cudaStream_t stream) {
    const TreePlan plan = plan_general(d);
    a.parts = plan.parts;
    a.part_tokens = plan.part_tokens;
    const int64_t all_rows = static_cast<int64_t>(a.batch) * a.kv_heads * a.rows;
    a.part_ml = reinterpret_cast<float2 *>(a.part_o);
    a.part_o += 2 * all_rows * plan.parts;
    int rc = launch_general<T>(a, plan, stream);
    if (rc != VKOP_OK || plan.parts == 1)
        return rc;
    tree_attention_join_kernel<T><<<static_cast<unsigned>((all_rows + kJoinWarps - 1) / kJoinWarps), kJoinWarps * 32, 0, stream>>>(a);
    note_launch();
    return check_launch();
}

int launch_tree_attention(const vkop_tree_attention_desc &d, const void *q, const void *k, const void *v, const int32_t *table,
                          const int32_t *context, const int32_t *parents, const int32_t *num_nodes, void *out, float *lse,
                          void *workspace, cudaStream_t stream) {
    if (d.batch == 0)
        return VKOP_OK;
    TreeArgs a;
    a.q = q;
    a.k = k;
    a.v = v;
    a.table = table;
    a.context = context;
    a.parents = parents;
    a.num_nodes = num_nodes;
    a.out = out;
    a.lse = lse;
    a.part_o = static_cast<float *>(workspace);
    a.num_pages = d.num_pages;
    a.table_stride = d.table_stride ? d.table_stride : d.max_pages;
    a.q_hs = d.q_head_stride ? d.q_head_stride : d.head_dim;
    a.q_ns = d.q_node_stride ? d.q_node_stride : a.q_hs * d.q_heads;
    a.q_bs = d.q_batch_stride ? d.q_batch_stride : a.q_ns * d.nodes;
    a.o_hs = d.out_head_stride ? d.out_head_stride : d.head_dim;
    a.o_ns = d.out_node_stride ? d.out_node_stride : a.o_hs * d.q_heads;
    a.o_bs = d.out_batch_stride ? d.out_batch_stride : a.o_ns * d.nodes;
    a.k_hs = d.k_head_stride ? d.k_head_stride : d.head_dim;
    a.k_ts = d.k_token_stride ? d.k_token_stride : a.k_hs * d.kv_heads;
    a.k_ps = d.k_page_stride ? d.k_page_stride : a.k_ts * d.page_size;
    a.v_hs = d.v_head_stride ? d.v_head_stride : d.head_dim;
    a.v_ts = d.v_token_stride ? d.v_token_stride : a.v_hs * d.kv_heads;
    a.v_ps = d.v_page_stride ? d.v_page_stride : a.v_ts * d.page_size;
    a.batch = static_cast<int>(d.batch);
    a.nodes = d.nodes;
    a.q_heads = d.q_heads;
    a.kv_heads = d.kv_heads;
    a.group = d.q_heads / d.kv_heads;
    a.head_dim = d.head_dim;
    a.page_size = d.page_size;
    a.max_pages = d.num_pages > 0 ? d.max_pages : 0;  // without pages the table is not looked at
    a.rows = d.nodes * a.group;
    a.scale_log2 = d.scale * kLog2e;
    // 16-byte pieces of rows: every pointer and stride a multiple of 8 elements
    int64_t bits = 0;
    for (const void *p : {q, k, v, static_cast<const void *>(out)})
        bits |= reinterpret_cast<intptr_t>(p) / 2;
    for (int64_t s : {a.q_bs, a.q_ns, a.q_hs, a.o_bs, a.o_ns, a.o_hs, a.k_ps, a.k_ts, a.k_hs, a.v_ps, a.v_ts, a.v_hs})
        bits |= s;
    if (tree_mma_serves(d) && bits % 8 == 0)
        return launch_tree_mma(a, d, workspace, stream);
    switch (d.dtype) {
    case VKOP_F32: return launch_t<float>(a, d, stream);
    case VKOP_F16: return launch_t<__half>(a, d, stream);
    case VKOP_BF16: return launch_t<__nv_bfloat16>(a, d, stream);
    default: return VKOP_INVALID_ARG;
    }
}

}  // namespace vkop_cuda
