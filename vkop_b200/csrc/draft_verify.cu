// Verification of a tree (or chain) of drafted tokens against the target's probabilities.
//
// One thread-block cluster serves one sequence, in one launch without scratch memory.
//
//  walk    The probabilities that the tests compare, p(parent)[token] and q(parent)[token], do not depend on the walk:
//          all nodes gather theirs at once.  One warp of every CTA then walks the tree on the copies in shared memory, all
//          with the same result, so no decision has to be handed between CTAs.  What is left of a node's distribution after
//          several rejections never has to be written down: max(max(p - c q, 0) / D - q, 0) = max(p - (c + D) q, 0) / D, so
//          one number c and the mass D describe it.
//  mass    Only where a second child of a node is tested after a rejection, D = sum max(p - c q, 0) takes a pass over the
//          vocabulary, and the last token takes one: every warp of the cluster sums a contiguous range of the row and stores
//          its sum into the shared memory of every CTA of the cluster, where one scan in a fixed order gives everybody the
//          total and the prefixes.
//  draw    The range in which the prefix sum passes u times the total is read once more (from L2) by the CTA that owns
//          it: each thread sums a short run, a scan finds the run, its thread walks it.
//
// All sums and comparisons are in 64 bits (the inputs are exact in them, c q loses at most 2^-53): a decision differs from
// that of any other 64-bit evaluation only where a random number lies within about 1e-15 of a border.
// Bound: the one row of p (and of q) per sequence that has to be read, and for few sequences the latency of the chain
// gather -> walk -> pass -> draw.
#include <cooperative_groups.h>

#include "common.cuh"
#include "launchers.h"

namespace vkop_cuda {

namespace cg = cooperative_groups;

constexpr int kVerifyThreads = 512;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kVerifyMaxCluster = 16;
constexpr int kVerifyPortableCluster = 8;

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

// An entry in 64 bits; negative and NaN ones, and those below the smallest normal 32-bit number, count as zero, infinity as
// 2^128.  Exact, and put together from the bits: the conversion instruction runs at an eighth of the rate of these
// operations and took a third of a pass.
// (16-bit entries have no bits for the low word.)
template <typename T>
__device__ __forceinline__ double prob64(float v) {
    const uint32_t u = __float_as_uint(v);
    const bool good = u - 0x00800000u <= 0x7F000000u;
    return __hiloint2double(good ? static_cast<int>((u >> 3) + 0x38000000u) : 0, good && sizeof(T) == 4 ? static_cast<int>(u << 29) : 0);
}

// The same where a zero may be 2^-127, with fewer operations: in p - c q with c >= 1 an entry p of zero leaves nothing either
// way, and 2^-127 in place of q = 0 is lost in the rounding.
template <typename T>
__device__ __forceinline__ double prob64_or_tiny(float v) {
    float x;
    asm("mul.ftz.f32 %0, %1, 0f3F800000;" : "=f"(x) : "f"(v));
    const uint32_t u = __float_as_uint(fmaxf(x, 0.0f));
    return __hiloint2double(static_cast<int>((u >> 3) + 0x38000000u), sizeof(T) == 4 ? static_cast<int>(u << 29) : 0);
}

template <typename T>
__device__ __forceinline__ double load_prob(const T *p) {
    return prob64<T>(Elem<T>::from_storage(*p));
}

// What is summed over a row: p, max(p - c q, 0), or p without the rejected tokens.
enum VerifyMass { kMassPlain = 0, kMassResidual = 1, kMassExcluded = 2 };

template <typename T>
struct RowMass {
    const T *p, *q;
    double c;
    VerifyMass mode;
    const int *gone;  // rejected tokens (kMassExcluded)
    int gone_count;

    __device__ __forceinline__ bool excluded(int64_t i) const {
        for (int j = 0; j < gone_count; j++)
            if (gone[j] == i)
                return true;
        return false;
    }
    __device__ __forceinline__ double weight(float pv, float qv) const {
        const double w = prob64_or_tiny<T>(pv) - c * prob64_or_tiny<T>(qv);
        return __double2hiint(w) < 0 ? 0.0 : w;
    }
    __device__ __forceinline__ double at(int64_t i) const {
        const float pv = Elem<T>::from_storage(p[i]);
        if (mode == kMassResidual)
            return weight(pv, Elem<T>::from_storage(q[i]));
        if (mode == kMassExcluded && excluded(i))
            return 0.0;
        return prob64<T>(pv);
    }
};

// Vectors 32 lanes apart from v0 on, `count` in all: 16 elements of each row in flight a lane.
template <typename T, bool RESIDUAL>
__device__ __forceinline__ double vector_mass(const T *p, const T *q, double c, int64_t count) {
    constexpr int VEC = Elem<T>::kPerVec, U = 16 / VEC;
    const uint4 *pv = reinterpret_cast<const uint4 *>(p), *qv = reinterpret_cast<const uint4 *>(q);
    double s[2] = {0.0, 0.0};
    for (int64_t v = threadIdx.x & 31; v < count; v += 32 * U) {
        uint4 x[U], y[U];
#pragma unroll
        for (int k = 0; k < U; k++) {
            x[k] = v + 32 * k < count ? load_stream(pv + v + 32 * k) : make_uint4(0, 0, 0, 0);
            if (RESIDUAL)
                y[k] = v + 32 * k < count ? load_stream(qv + v + 32 * k) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < U; k++) {
            float f[VEC], g[VEC];
            Elem<T>::unpack(x[k], f);
            if (RESIDUAL)
                Elem<T>::unpack(y[k], g);
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                if (RESIDUAL) {
                    const double w = prob64_or_tiny<T>(f[e]) - c * prob64_or_tiny<T>(g[e]);
                    if (__double2hiint(w) >= 0)
                        s[e & 1] += w;
                } else {
                    s[e & 1] += prob64<T>(f[e]);
                }
            }
        }
    }
    return s[0] + s[1];
}

// Sum over [lo, hi), which a warp reads together; p + vlo is 16-byte aligned.
template <typename T>
__device__ double warp_range_mass(const RowMass<T> &m, int64_t lo, int64_t hi, int64_t vlo, bool q_aligned) {
    constexpr int VEC = Elem<T>::kPerVec;
    const int lane = threadIdx.x & 31;
    // few ranges hold a rejected token: only those look at the list, an element at a time; so do rows of p and q that lie
    // differently on the 16-byte boundaries
    bool slow = m.mode == kMassResidual && !q_aligned;
    if (m.mode == kMassExcluded) {
        bool look = false;
        for (int j = lane; j < m.gone_count; j += 32)
            look |= m.gone[j] >= lo && m.gone[j] < hi;
        slow = __any_sync(kFullMask, look);
    }
    const int64_t start = max(lo, vlo);
    const int64_t count = !slow && start < hi ? (hi - start) / VEC : 0, from = start + count * VEC;
    double s = 0.0;
    if (count > 0)
        s = m.mode == kMassResidual ? vector_mass<T, true>(m.p + start, m.q + start, m.c, count) : vector_mass<T, false>(m.p + start, nullptr, 0.0, count);
    for (int64_t i = lo + lane; i < min(start, hi); i += 32)  // in front of the first aligned vector
        s += m.at(i);
    for (int64_t i = from + lane; i < hi; i += 32)  // behind the last one
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
    double *s_q = s_p + N;                           // [N] the draft's; 1 where the token was certain
    double *s_uq = s_q + N;                          // [N] its random number times that
    double *s_left = s_uq + N, *s_of = s_left + N;   // [N] the two sides of a test without the random number; 0 of 0: not tested
    int *s_par = reinterpret_cast<int *>(s_of + N);  // -1: nobody's child
    int *s_tok = s_par + N;
    int *s_path = s_tok + N, *s_gone = s_path + N;
    __shared__ double s_all[2][kVerifyMaxCluster * kVerifyWarps * 9 / 8];  // sums of the cluster's warps, by pass parity
    __shared__ double s_scan[kVerifyWarps];
    __shared__ int s_last, s_found, s_gone_count;

    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // waited for before the first store to another CTA

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
        s_p[i] = ok ? load_prob(target + par * a.target_ns + tok) : 0.0;
        s_q[i] = ok && par < a.draft_rows ? load_prob(draft + par * a.draft_ns + tok) : 1.0;
        s_par[i] = ok ? par : -1;
        s_tok[i] = ok ? static_cast<int>(tok) : -1;
        s_uq[i] = static_cast<double>(a.u[b * N + i]) * s_q[i];
        s_left[i] = 0.0;
        s_of[i] = 0.0;
        s_path[i] = i == 0 && used > 0 ? 0 : -1;
    }
    __syncthreads();

    constexpr int VEC = Elem<T>::kPerVec;
    constexpr int PER_LANE = kVerifyMaxCluster * kVerifyWarps / 32;  // ranges that a lane scans, at most
    const int ranges = csize * kVerifyWarps, per_lane = (ranges + 31) / 32;
    auto place = [](int r) { return r + (r >> 3); };  // padded: the lanes' reads fall on different banks
    const int64_t width = ((a.vocab + ranges - 1) / ranges + VEC - 1) / VEC * VEC;
    auto head_of = [&](const T *row) { return static_cast<int64_t>(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T)); };
    auto range_lo = [&](int64_t head, int r) { return r == 0 ? 0 : min(a.vocab, head + r * width); };
    int passes = 0;
    // The sum of one pass over a row, the same bits in every thread of the cluster.  Given an aim, as a share of the total:
    // *own the range in which the prefix sum passes it, *before the prefix in front of that range.  By rounding, or for a
    // share >= 1, none may: then the last range that holds anything.
    auto cluster_mass = [&](const RowMass<T> &m, double share, int *own, double *before, double *aim) {
        const int mine = rank * kVerifyWarps + warp;
        const int64_t head = head_of(m.p);
        const bool q_aligned = (reinterpret_cast<uintptr_t>(m.q) & 15) == (reinterpret_cast<uintptr_t>(m.p) & 15);
        const double s = warp_range_mass<T>(m, range_lo(head, mine), min(a.vocab, head + (mine + 1) * width), head, q_aligned);
        double *all = s_all[passes & 1];
        if (passes == 0)
            asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // all CTAs of the cluster run
        if (lane < csize)
            *cluster.map_shared_rank(&all[place(mine)], lane) = s;
        cluster.sync();  // (a pass apart, so that nobody still reads what the pass after the next one writes)
        passes++;
        double v[PER_LANE], sum = 0.0;
#pragma unroll
        for (int k = 0; k < PER_LANE; k++) {
            v[k] = 0.0;
            if (k < per_lane && lane * per_lane + k < ranges)
                v[k] = all[place(lane * per_lane + k)];
            sum += v[k];
        }
        double upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(kFullMask, upto, o);
            upto += lane >= o ? y : 0.0;
        }
        const double total = __shfl_sync(kFullMask, upto, 31);
        if (own) {
            *aim = share * total;
            double run = __shfl_up_sync(kFullMask, upto, 1);
            run = lane == 0 ? 0.0 : run;
            int at = -1;
            double at_before = 0.0;
#pragma unroll
            for (int k = 0; k < PER_LANE; k++) {
                if (at < 0 && run + v[k] > *aim) {
                    at = lane * per_lane + k;
                    at_before = run;
                }
                run += v[k];
            }
            unsigned hit = __ballot_sync(kFullMask, at >= 0);
            int who = __ffs(hit) - 1;
            if (hit == 0) {
                run = upto - sum;
#pragma unroll
                for (int k = 0; k < PER_LANE; k++) {
                    if (v[k] > 0.0) {
                        at = lane * per_lane + k;
                        at_before = run;
                    }
                    run += v[k];
                }
                hit = __ballot_sync(kFullMask, at >= 0);
                who = 31 - __clz(hit);  // -1 for an empty row: nothing is drawn then
            }
            *own = __shfl_sync(kFullMask, at, who & 31);
            *before = __shfl_sync(kFullMask, at_before, who & 31);
        }
        return total;
    };

    // ---- walk ----
    __shared__ double s_c;
    __shared__ int s_cur, s_count, s_stale, s_need;
    int cur = 0, last = 0, count = used > 0 ? 1 : 0;
    double c = 0.0, mass = 1.0;
    bool stale = false;  // c has grown, mass not yet taken
    RowMass<T> m{target, draft, 0.0, kMassPlain, s_gone, 0};
    while (true) {
        if (warp == 0) {  // until it ends or a mass is needed
            int need = 0;
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
                    need = 1;
                    break;
                }
                double left = s_p[child];
                if (drawn) {
                    const double w = left - c * s_q[child];
                    left = w > 0.0 ? w : 0.0;
                } else {  // a token that was rejected before has nothing left
                    const int tok = s_tok[child];
                    bool again = false;
                    for (int base = 0; base < child; base += 32) {
                        const int i = base + lane;
                        again |= __ballot_sync(kFullMask, i > 0 && i < child && s_par[i] == cur && s_tok[i] == tok) != 0;
                    }
                    left = again ? 0.0 : left;
                }
                const bool took = mass * s_uq[child] < left;
                if (lane == 0) {
                    s_left[child] = left;
                    s_of[child] = mass * s_q[child];
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
            if (lane == 0)
                s_cur = cur, s_count = count, s_stale = stale, s_need = need, s_c = c;
        }
        __syncthreads();
        cur = s_cur;
        count = s_count;
        stale = s_stale != 0;
        c = s_c;
        if (!s_need)
            break;
        m.p = target + cur * a.target_ns;
        m.q = draft + cur * a.draft_ns;
        m.c = c;
        m.mode = kMassResidual;
        mass = cluster_mass(m, 0.0, nullptr, nullptr, nullptr);  // (ends behind a barrier: the state may be written again)
        stale = false;
    }

    if (rank == 0) {
        for (int i = tid; i < N; i += kVerifyThreads) {
            a.out_path[b * N + i] = s_path[i];
            if (a.out_chance)
                a.out_chance[b * N + i] = s_left[i] >= s_of[i] ? (s_left[i] > 0.0 ? 1.0f : 0.0f) : static_cast<float>(s_left[i] / s_of[i]);
        }
        if (tid == 0)
            a.out_count[b] = count;
    }

    // ---- draw ----
    int64_t token = -1;
    if (used > 0) {
        m.p = target + cur * a.target_ns;
        m.q = draft + cur * a.draft_ns;
        m.c = c;
        m.mode = kMassPlain;
        if (stale) {
            m.mode = kMassResidual;
        } else if (cur >= a.draft_rows) {  // the walk ended here: every child was tested and rejected
            if (tid == 0)
                s_gone_count = 0;
            __syncthreads();
            for (int i = tid; i < used; i += kVerifyThreads)
                if (s_par[i] == cur)
                    s_gone[atomicAdd(&s_gone_count, 1)] = s_tok[i];  // in any order
            __syncthreads();
            m.gone_count = s_gone_count;
            if (m.gone_count > 0)
                m.mode = kMassExcluded;
        }
        int own = -1;
        double before = 0.0, aim = 0.0;
        double total = cluster_mass(m, s_uq[0], &own, &before, &aim);
        if (!(total > 0.0) && m.mode != kMassPlain) {
            m.mode = kMassPlain;  // nothing left: the distribution itself
            total = cluster_mass(m, s_uq[0], &own, &before, &aim);
        }
        if (total > 0.0) {
            if (own / kVerifyWarps == rank) {
                const int64_t head = head_of(m.p), lo = range_lo(head, own), hi = min(a.vocab, head + (own + 1) * width);
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
}

template <typename T>
static int launch_draft_verify_t(const vkop_draft_verify_desc &d, const VerifyArgs &a, cudaStream_t stream) {
    // CTAs for two on every SM, as long as a warp's range stays a few vectors long; clusters beyond the portable size where
    // the GPCs hold them all (one sequence over 128256 f32 columns: 9.4 us against 10.1 with 8, 16 trees drawn over 256000 bf16
    // columns: 28.5 us against 34.5)
    int csize = 1;
    const int most = d.batch <= 16 ? kVerifyMaxCluster : kVerifyPortableCluster;
    while (csize < most && d.batch * csize * 2 <= 2 * 148 && d.vocab / (csize * 2) >= 2048)
        csize *= 2;
    const size_t smem = static_cast<size_t>(d.nodes) * (5 * sizeof(double) + 4 * 4);
    if (smem > 32 * 1024 && cudaFuncSetAttribute(draft_verify_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess) {
        cudaGetLastError();
        return VKOP_CUDA_ERROR;
    }
    if (csize > kVerifyPortableCluster && cudaFuncSetAttribute(draft_verify_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
        cudaGetLastError();
        csize = kVerifyPortableCluster;
    }
    while (true) {
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
        if (cudaLaunchKernelEx(&cfg, draft_verify_kernel<T>, a) == cudaSuccess)
            break;
        cudaGetLastError();
        if (csize <= kVerifyPortableCluster)
            return VKOP_CUDA_ERROR;
        csize = kVerifyPortableCluster;  // no place for the larger cluster here (a part of a GPU)
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
