// Verification of a tree (or chain) of drafted tokens against the target's probabilities.
//
// One thread-block cluster serves one sequence, in one launch without scratch memory.
//
//  walk    The probabilities that the tests compare, p(parent)[token] and q(parent)[token], do not depend on the walk:
//          all nodes gather theirs at once.  Every warp of the cluster then walks the tree on the copies in shared memory,
//          all with the same result, so no decision has to be handed around.  What is left of a node's distribution after
//          several rejections never has to be written down: max(max(p - c q, 0) / D - q, 0) = max(p - (c + D) q, 0) / D, so
//          one number c and the mass D describe it.
//  mass    Only where a second child of a node is tested after a rejection, D = sum max(p - c q, 0) takes a pass over the
//          vocabulary, and the last token takes one: every warp of the cluster sums a contiguous range of the row, the
//          sums are read through distributed shared memory and added in one fixed order by everybody.
//  draw    The range in which the prefix sum passes u times the total is read once more (from L2) by the CTA that owns
//          it: each thread sums a short run, a scan finds the run, its thread walks it.
//
// All sums and comparisons are in 64 bits (the inputs are exact in them, c q loses at most 2^-53): a decision differs from
// that of any other 64-bit evaluation only where a random number lies within about 1e-15 of a border.
// Bound: the one row of p (and of q) per sequence that has to be read, and for few sequences the latency of the chain
// gather -> walk -> pass -> draw.
#include <cfloat>

#include <cooperative_groups.h>

#include "common.cuh"
#include "launchers.h"

namespace vkop_cuda {

namespace cg = cooperative_groups;

constexpr int kVerifyThreads = 512;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kVerifyMaxCluster = 8;  // portable cluster size
constexpr int kExcludeBuckets = 8192;  // hash of 8-element groups that hold a rejected token (certain drafts)

struct VerifyArgs {
    const void *target, *draft, *tokens;
    const int32_t *parents, *num_nodes;
    const float *u;
    int32_t *out_path, *out_count;
    void *out_token;
    float *out_chance;
    int64_t vocab, target_bs, target_ns, draft_bs, draft_ns;
    int nodes, draft_rows, index_dtype;
};

// negative, NaN and infinite entries count as zero
__device__ __forceinline__ float clean_prob(float v) { return (v > 0.0f && v <= FLT_MAX) ? v : 0.0f; }

template <typename T>
__device__ __forceinline__ float load_prob(const T *p) {
    return clean_prob(Elem<T>::from_storage(*p));
}

// What is summed over a row: p, max(p - c q, 0), or p without the rejected tokens.
enum VerifyMass { kMassPlain = 0, kMassResidual = 1, kMassExcluded = 2 };

template <typename T>
struct RowMass {
    const T *p, *q;
    double c;
    VerifyMass mode;
    // rejected tokens (kMassExcluded): children of `cur` below `until`
    const int *par, *tok;
    const uint32_t *buckets;
    int cur, until;

    __device__ __forceinline__ bool excluded(int64_t i) const {
        const uint32_t h = static_cast<uint32_t>(i >> 3) % kExcludeBuckets;
        if (!(buckets[h >> 5] >> (h & 31) & 1u))
            return false;
        for (int j = 1; j < until; j++)
            if (par[j] == cur && tok[j] == i)
                return true;
        return false;
    }
    __device__ __forceinline__ double weight(float pv, float qv) const {
        const double w = static_cast<double>(clean_prob(pv)) - c * static_cast<double>(clean_prob(qv));
        return w > 0.0 ? w : 0.0;
    }
    __device__ __forceinline__ double at(int64_t i) const {
        const float pv = Elem<T>::from_storage(p[i]);
        if (mode == kMassResidual)
            return weight(pv, Elem<T>::from_storage(q[i]));
        if (mode == kMassExcluded && excluded(i))
            return 0.0;
        return static_cast<double>(clean_prob(pv));
    }
};

// Sum over [lo, hi), which a warp reads together; (p + vlo) is 16-byte aligned for the vector part [vlo, vhi).
template <typename T>
__device__ double warp_range_mass(const RowMass<T> &m, int64_t lo, int64_t hi, int64_t vlo, bool q_aligned) {
    constexpr int VEC = Elem<T>::kPerVec, U = 4;
    const int lane = threadIdx.x & 31;
    double s = 0.0;
    if (lo < vlo) {  // the part in front of the first aligned vector: fewer than VEC elements
        const int64_t i = lo + lane;
        if (i < min(vlo, hi))
            s += m.at(i);
    }
    const int64_t start = max(lo, vlo);
    const int64_t nvec = start < hi ? (hi - start) / VEC : 0;
    for (int64_t v = lane; v < nvec; v += 32 * U) {
        uint4 pv[U], qv[U];
#pragma unroll
        for (int k = 0; k < U; k++)
            if (v + 32 * k < nvec)
                pv[k] = load_stream(reinterpret_cast<const uint4 *>(m.p + start) + v + 32 * k);
        if (m.mode == kMassResidual && q_aligned) {
#pragma unroll
            for (int k = 0; k < U; k++)
                if (v + 32 * k < nvec)
                    qv[k] = load_stream(reinterpret_cast<const uint4 *>(m.q + start) + v + 32 * k);
        }
#pragma unroll
        for (int k = 0; k < U; k++) {
            if (v + 32 * k >= nvec)
                break;
            const int64_t i0 = start + (v + 32 * k) * VEC;
            float f[VEC];
            Elem<T>::unpack(pv[k], f);
            if (m.mode == kMassResidual) {
                float g[VEC];
                if (q_aligned) {
                    Elem<T>::unpack(qv[k], g);
                } else {
#pragma unroll
                    for (int e = 0; e < VEC; e++)
                        g[e] = Elem<T>::from_storage(m.q[i0 + e]);
                }
#pragma unroll
                for (int e = 0; e < VEC; e++)
                    s += m.weight(f[e], g[e]);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; e++)
                    s += (m.mode == kMassExcluded && m.excluded(i0 + e)) ? 0.0 : static_cast<double>(clean_prob(f[e]));
            }
        }
    }
    const int64_t i = start + nvec * VEC + lane;  // fewer than VEC elements behind the last vector
    if (start < hi && i < hi)
        s += m.at(i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        s += __shfl_xor_sync(kFullMask, s, o);
    return s;
}

template <typename T>
__global__ void __launch_bounds__(kVerifyThreads, 2) draft_verify_kernel(const VerifyArgs a) {
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = static_cast<int>(cluster.block_rank()), csize = static_cast<int>(cluster.num_blocks());
    const int64_t b = blockIdx.x / csize;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int N = a.nodes;

    extern __shared__ __align__(16) unsigned char smem[];
    double *s_p = reinterpret_cast<double *>(smem);  // [N] target probability of a node's token at its parent
    double *s_q = s_p + N;                           // [N] the draft's
    float *s_u = reinterpret_cast<float *>(s_q + N);
    float *s_chance = s_u + N;
    int *s_par = reinterpret_cast<int *>(s_chance + N);  // -1: nobody's child
    int *s_tok = s_par + N;
    int *s_path = s_tok + N;
    __shared__ double s_sum[2][kVerifyWarps];                       // this CTA's warp sums, by pass parity (read by the cluster)
    __shared__ double s_all[kVerifyMaxCluster * kVerifyWarps];      // everybody's
    __shared__ double s_scan[kVerifyWarps];
    __shared__ uint32_t s_buckets[kExcludeBuckets / 32];
    __shared__ int s_last, s_found;

    int used = N;
    if (a.num_nodes)
        used = min(max(a.num_nodes[b], 0), N);
    const T *target = static_cast<const T *>(a.target) + b * a.target_bs;
    const T *draft = static_cast<const T *>(a.draft) + b * a.draft_bs;
    for (int i = tid; i < N; i += kVerifyThreads) {
        const int par = a.parents ? a.parents[b * N + i] : i - 1;
        const int64_t tok = a.index_dtype == VKOP_I64 ? static_cast<const int64_t *>(a.tokens)[b * N + i]
                                                      : static_cast<const int32_t *>(a.tokens)[b * N + i];
        const bool ok = i > 0 && i < used && par >= 0 && par < i && tok >= 0 && tok < a.vocab;
        s_p[i] = ok ? static_cast<double>(load_prob(target + par * a.target_ns + tok)) : 0.0;
        s_q[i] = ok && par < a.draft_rows ? static_cast<double>(load_prob(draft + par * a.draft_ns + tok)) : 1.0;
        s_par[i] = ok ? par : -1;
        s_tok[i] = ok ? static_cast<int>(tok) : -1;
        s_u[i] = a.u[b * N + i];
        s_chance[i] = 0.0f;
        s_path[i] = i == 0 && used > 0 ? 0 : -1;
    }
    __syncthreads();

    int passes = 0;
    // the sum of one pass, the same bits in every thread of the cluster; s_all keeps the sums of the ranges in row order
    auto cluster_mass = [&](const RowMass<T> &m) {
        constexpr int VEC = Elem<T>::kPerVec;
        const int ranges = csize * kVerifyWarps, mine = rank * kVerifyWarps + warp;
        const int64_t head = ((16 - (reinterpret_cast<uintptr_t>(m.p) & 15)) & 15) / sizeof(T);
        const int64_t width = ((a.vocab + ranges - 1) / ranges + VEC - 1) / VEC * VEC;
        const int64_t lo = mine == 0 ? 0 : min(a.vocab, head + mine * width), hi = min(a.vocab, head + (mine + 1) * width);
        const bool q_aligned = (reinterpret_cast<uintptr_t>(m.q) & 15) == (reinterpret_cast<uintptr_t>(m.p) & 15);
        const double s = warp_range_mass<T>(m, lo, hi, head, q_aligned);
        if (lane == 0)
            s_sum[passes & 1][warp] = s;
        cluster.sync();
        if (tid < ranges)
            s_all[tid] = *cluster.map_shared_rank(&s_sum[passes & 1][tid % kVerifyWarps], tid / kVerifyWarps);
        __syncthreads();
        passes++;
        double t = 0.0;
        for (int k = 0; k < ranges; k += 32) {
            double x = k + lane < ranges ? s_all[k + lane] : 0.0;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1)
                x += __shfl_xor_sync(kFullMask, x, o);
            t += x;
        }
        return t;
    };

    // ---- walk ----
    int cur = 0, last = 0, count = used > 0 ? 1 : 0;
    double c = 0.0, mass = 1.0;
    bool stale = false;  // c has grown, mass not yet taken
    RowMass<T> m{target, draft, 0.0, kMassPlain, s_par, s_tok, s_buckets, 0, 0};
    while (true) {
        int child = 0;
        for (int base = (last + 1) & ~31; base < used && child == 0; base += 32) {
            const int i = base + lane;
            const unsigned hit = __ballot_sync(kFullMask, i > last && i < used && s_par[i] == cur);
            if (hit)
                child = base + __ffs(hit) - 1;
        }
        if (child == 0)
            break;
        const bool drawn = cur < a.draft_rows;
        if (stale) {
            m.p = target + cur * a.target_ns;
            m.q = draft + cur * a.draft_ns;
            m.c = c;
            m.mode = kMassResidual;
            mass = cluster_mass(m);
            stale = false;
        }
        double left = s_p[child], scaled = mass;
        if (drawn) {
            const double w = left - c * s_q[child];
            left = w > 0.0 ? w : 0.0;
            scaled = mass * s_q[child];
        } else {  // a token that was rejected before has nothing left
            const int tok = s_tok[child];
            bool again = false;
            for (int base = 0; base < child; base += 32) {
                const int i = base + lane;
                again |= __ballot_sync(kFullMask, i > 0 && i < child && s_par[i] == cur && s_tok[i] == tok) != 0;
            }
            left = again ? 0.0 : left;
        }
        const bool took = static_cast<double>(s_u[child]) * scaled < left;
        if (tid == 0) {
            s_chance[child] = left >= scaled ? (left > 0.0 ? 1.0f : 0.0f) : static_cast<float>(left / scaled);
            if (took)
                s_path[count] = child;
        }
        if (took) {
            cur = child;
            count++;
            c = 0.0;
            mass = 1.0;
        } else if (drawn) {
            c += mass;
            stale = true;
        } else {
            mass = mass > left ? mass - left : 0.0;
        }
        last = child;
    }

    // ---- draw ----
    int64_t token = -1;
    if (used > 0) {
        m.p = target + cur * a.target_ns;
        m.q = draft + cur * a.draft_ns;
        m.c = c;
        m.cur = cur;
        m.until = used;
        m.mode = kMassPlain;
        if (stale) {
            m.mode = kMassResidual;
        } else if (cur >= a.draft_rows) {  // the walk ended here: every child was tested and rejected
            bool any = false;
            for (int i = tid; i < used; i += kVerifyThreads)
                any |= s_par[i] == cur;
            if (__syncthreads_or(any))
                m.mode = kMassExcluded;
        }
        if (m.mode == kMassExcluded) {
            for (int i = tid; i < kExcludeBuckets / 32; i += kVerifyThreads)
                s_buckets[i] = 0;
            __syncthreads();
            for (int i = tid; i < used; i += kVerifyThreads)
                if (s_par[i] == cur) {
                    const uint32_t h = static_cast<uint32_t>(s_tok[i] >> 3) % kExcludeBuckets;
                    atomicOr(&s_buckets[h >> 5], 1u << (h & 31));
                }
            __syncthreads();
        }
        double total = cluster_mass(m);
        if (!(total > 0.0) && m.mode != kMassPlain) {
            m.mode = kMassPlain;  // nothing left: the distribution itself
            total = cluster_mass(m);
        }
        if (total > 0.0) {
            const int ranges = csize * kVerifyWarps;
            const double aim = static_cast<double>(s_u[0]) * total;
            // the range where the prefix sum passes the aim; by rounding or a number >= 1 none may: then the last that holds anything
            int own = -1, full = 0;
            double before = 0.0, run = 0.0, full_before = 0.0;
            for (int k = 0; k < ranges && own < 0; k++) {
                if (s_all[k] > 0.0) {
                    full = k;
                    full_before = run;
                }
                if (run + s_all[k] > aim) {
                    own = k;
                    before = run;
                }
                run += s_all[k];
            }
            if (own < 0) {
                own = full;
                before = full_before;
            }
            if (own / kVerifyWarps == rank) {
                constexpr int VEC = Elem<T>::kPerVec;
                const int64_t head = ((16 - (reinterpret_cast<uintptr_t>(m.p) & 15)) & 15) / sizeof(T);
                const int64_t width = ((a.vocab + ranges - 1) / ranges + VEC - 1) / VEC * VEC;
                const int64_t lo = own == 0 ? 0 : min(a.vocab, head + own * width), hi = min(a.vocab, head + (own + 1) * width);
                const int64_t per = (hi - lo + kVerifyThreads - 1) / kVerifyThreads;
                const int64_t from = min(hi, lo + tid * per), to = min(hi, from + per);
                double sum = 0.0;
                int some = -1;  // this thread's last element that holds anything, from `lo`
                for (int64_t i = from; i < to; i++) {
                    const double w = m.at(i);
                    sum += w;
                    if (w > 0.0)
                        some = static_cast<int>(i - lo);
                }
                double upto = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double x = __shfl_up_sync(kFullMask, upto, o);
                    upto += lane >= o ? x : 0.0;
                }
                if (lane == 31)
                    s_scan[warp] = upto;
                if (tid == 0)
                    s_last = -1, s_found = kVerifyThreads;
                __syncthreads();
                for (int w = 0; w < warp; w++)
                    before += s_scan[w];
                if (some >= 0) {
                    atomicMax(&s_last, some);
                    if (before + upto > aim)
                        atomicMin(&s_found, tid);
                }
                __syncthreads();
                const int who = s_found;
                if (who == kVerifyThreads) {
                    token = lo + s_last;
                } else if (tid == who) {
                    double r = before + (upto - sum);
                    token = lo + some;
                    for (int64_t i = from; i < to; i++) {
                        r += m.at(i);
                        if (r > aim) {
                            token = i;
                            break;
                        }
                    }
                }
                if (tid == (who == kVerifyThreads ? 0 : who))
                    store_index(a.out_token, a.index_dtype, b, token);
            }
        } else if (rank == 0 && tid == 0) {
            store_index(a.out_token, a.index_dtype, b, -1);
        }
    } else if (rank == 0 && tid == 0) {
        store_index(a.out_token, a.index_dtype, b, -1);
    }

    if (rank == 0) {
        __syncthreads();  // thread 0's entries of the path
        for (int i = tid; i < N; i += kVerifyThreads) {
            a.out_path[b * N + i] = s_path[i];
            if (a.out_chance)
                a.out_chance[b * N + i] = s_chance[i];
        }
        if (tid == 0)
            a.out_count[b] = count;
    }
    if (passes > 0)
        cluster.sync();  // no CTA leaves while another may still read its sums
}

template <typename T>
static int launch_draft_verify_t(const vkop_draft_verify_desc &d, const VerifyArgs &a, cudaStream_t stream) {
    // CTAs for two on every SM, as long as a warp's range stays a few vectors long
    int csize = 1;
    while (csize < kVerifyMaxCluster && d.batch * csize * 2 <= 2 * 148 && d.vocab / (csize * 2) >= 2048)
        csize *= 2;
    const size_t smem = static_cast<size_t>(d.nodes) * (2 * sizeof(double) + 5 * 4);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(d.batch * csize));
    cfg.blockDim = dim3(kVerifyThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(csize);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, draft_verify_kernel<T>, a) != cudaSuccess) {
        cudaGetLastError();
        return VKOP_CUDA_ERROR;
    }
    note_launch();
    return VKOP_OK;
}

int launch_draft_verify(const vkop_draft_verify_desc &d, const void *target, const void *draft, const void *tokens,
                        const int32_t *parents, const int32_t *num_nodes, const float *u, int32_t *out_path, int32_t *out_count,
                        void *out_token, float *out_chance, cudaStream_t stream) {
    if (d.batch == 0)
        return VKOP_OK;
    VerifyArgs a;
    a.target = target;
    a.draft = draft;
    a.tokens = tokens;
    a.parents = parents;
    a.num_nodes = num_nodes;
    a.u = u;
    a.out_path = out_path;
    a.out_count = out_count;
    a.out_token = out_token;
    a.out_chance = out_chance;
    a.vocab = d.vocab;
    a.target_ns = d.target_node_stride ? d.target_node_stride : d.vocab;
    a.target_bs = d.target_batch_stride ? d.target_batch_stride : a.target_ns * d.nodes;
    a.draft_ns = d.draft_node_stride ? d.draft_node_stride : d.vocab;
    a.draft_bs = d.draft_batch_stride ? d.draft_batch_stride : a.draft_ns * d.draft_rows;
    a.nodes = d.nodes;
    a.draft_rows = draft ? d.draft_rows : 0;
    a.index_dtype = d.index_dtype;
    switch (d.dtype) {
    case VKOP_F32: return launch_draft_verify_t<float>(d, a, stream);
    case VKOP_F16: return launch_draft_verify_t<__half>(d, a, stream);
    case VKOP_BF16: return launch_draft_verify_t<__nv_bfloat16>(d, a, stream);
    default: return VKOP_INVALID_ARG;
    }
}

}  // namespace vkop_cuda
