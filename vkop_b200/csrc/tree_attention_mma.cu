// Attention of a tree of drafted tokens over a paged cache on the tensor cores: 16-bit types, head sizes 64 and 128.
//
// The rows that share a cache head (nodes x query heads a cache head) fill the M dimension of 128-row products; a tile of 128
// cached positions is the N dimension of S = Q K^T and the K dimension of O += P V.  Roles of a CTA (one a SM, 16 warps):
//   warps 0-7    softmax: two groups of 128 threads, a thread a row.  With more than 128 rows each group has its own 128 and
//                both see every tile (ROWT = 2); otherwise the groups take the tiles in turn and their sums are joined at the
//                end (ROWT = 1), so that one group's exponentials overlap the other's products either way.
//   warps 8-11   copies: 16-byte asynchronous copies gather the rows of a tile from their pages into a ring of buffers in the
//                128-byte swizzled layout that the products read (any page size, any strides; rows past the end become zeros).
//   warp 12      one thread issues the products; S (then P in its place) and O live in tensor memory.
//
// S: exponents are taken relative to a reference that follows the row's maximum only when it grows by more than 2^8 (the sums
// are rescaled then, in tensor memory); P is scaled by 2^kBias so that 16-bit weights stay clear of the subnormal range.
//
// Work is cut without regard to sequence borders: all tiles of the call, sequence by sequence, head by head, are one list that
// the CTAs share out evenly, whatever the lengths of the sequences.  A (sequence, head, rows) unit that one CTA holds entirely
// is written out; of others every CTA leaves its part in its own two slots of the scratch memory (first and last unit of its
// range) and the join adds them up.
//
// Bound: reading the cache once from HBM for few rows a head; around 256 rows the products and the exponentials
// (16 a clock and SM) take as long as the copies.
#include "tensor_core.cuh"
#include "tree_attention.cuh"

namespace vkop_cuda {

constexpr int kMmaThreads = 512;
constexpr int kTile = 128;       // positions a tile
constexpr int kMmaCtas = 148;
constexpr float kBias = 6.0f;    // log2 of the scale of the weights
constexpr float kGrow = 8.0f;    // log2 of the growth of the maximum that is let pass; 2^(6 + 8) < 65504
constexpr int kSlots = 8;        // tiles (and units) whose flags may be alive at once: more than a ring holds

struct TreeMmaArgs {
    TreeArgs a;
    int64_t *starts;  // [batch + 1] first tile of a sequence in the list of all tiles
    int mtiles;       // groups of ROWT * 128 rows a head
    float scale;      // |scale| * log2(e)
    uint32_t flip;    // sign bits of two elements when the scale is negative: the queries take the sign
    uint32_t mask;    // 0 when the scale is 0: so do they then (masked scores are -inf, which 0 cannot scale)
};

template <int D, int ROWT>
struct TreeMmaShape {
    static constexpr int kBuffer = kTile * D * 2;
    static constexpr int kRing = D == 128 ? (ROWT == 2 ? 5 : 6) : 8;
    static constexpr int kQ = ROWT * 128 * D * 2;
    static constexpr int kExtras = 3072;
    static constexpr int kSmem = kQ + kRing * kBuffer + kExtras;
};

struct TreeMmaExtras {
    uint64_t full[8], empty[8], s_ready[2], p_ready[2], pv_done[2], q_ready;
    int64_t left;
    uint32_t tmem;
    int abort, begin_b, begin_u, begin_j, pad;
    alignas(16) uint32_t valid[kSlots][4];
    int bad[kSlots];
    uint8_t parents[2][kTreeMaxNodes];
    float2 ml[2][128];
};
static_assert(sizeof(TreeMmaExtras) <= 3072, "extras");

__device__ __forceinline__ int tree_tiles(const TreeArgs &a, int b) {
    const int64_t length = tree_context(a, b) + tree_used(a, b);
    return length <= 0 ? 1 : static_cast<int>((length + kTile - 1) / kTile);
}

// The units that a CTA's range of tiles runs through.
struct TreeWalk {
    int64_t left;
    int b, u, j0, j1, tiles, seg;
    int64_t context, length;
    int used;
    __device__ __forceinline__ void begin(const TreeMmaExtras &x) {
        left = x.left;
        b = x.begin_b;
        u = x.begin_u;
        j1 = x.begin_j;
        seg = -1;
        tiles = -1;
    }
    __device__ __forceinline__ bool next(const TreeArgs &a, int units) {
        if (left <= 0)
            return false;
        if (tiles >= 0 && j1 == tiles) {
            j1 = 0;
            if (++u == units) {
                u = 0;
                b++;
                tiles = -1;
            }
        }
        if (tiles < 0) {
            context = tree_context(a, b);
            used = tree_used(a, b);
            length = context + used;
            tiles = length <= 0 ? 1 : static_cast<int>((length + kTile - 1) / kTile);
        }
        j0 = j1;
        j1 = left < tiles - j0 ? j0 + static_cast<int>(left) : tiles;
        left -= j1 - j0;
        seg++;
        return true;
    }
    __device__ __forceinline__ bool whole() const { return j0 == 0 && j1 == tiles; }
};

template <int N>
__device__ __forceinline__ void set_registers_up() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void set_registers_down() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// ---- copies ----
template <typename T, int D, int ROWT>
__device__ __forceinline__ void tree_copy_role(const TreeMmaArgs &g, TreeMmaExtras &x, uint32_t ring, int units) {
    using Shape = TreeMmaShape<D, ROWT>;
    constexpr int NB = Shape::kRing;
    constexpr int CHUNKS = D / 8;          // 16-byte pieces of a row
    constexpr int ROWS = 32 / CHUNKS;      // rows a warp copies at a time
    const TreeArgs &a = g.a;
    const int lane = threadIdx.x & 31, pw = (threadIdx.x >> 5) & 3;
    const int chunk = lane % CHUNKS, sub = lane / CHUNKS;
    const uint32_t column = static_cast<uint32_t>(chunk >> 3) * (kTile * 128);
    volatile int *abort = &x.abort;
    int next = 0;                // buffers issued so far
    int told = 0;                // buffers announced so far: next - told <= 2 between calls
    // a value tile with drafted rows: their values that are not finite are taken out (the epilogue adds them to the rows that
    // attend them; as a factor of a zero weight they would spoil the others)
    int64_t check_from = 0;      // first drafted row of the tile in question, in rows of this warp
    int check_buffer = -1, check_seg = 0;
    auto announce = [&](int upto) {
        for (; told < upto; told++) {
            const uint32_t buf = ring + static_cast<uint32_t>(told % NB) * Shape::kBuffer;
            if (told == check_buffer) {
#pragma unroll 1
                for (int i = 0; i < 32 / ROWS; i++) {
                    const int r = sub + i * ROWS;
                    if (r < check_from)
                        continue;
                    const uint32_t at = buf + column + static_cast<uint32_t>(pw * 32 + r) * 128 + (static_cast<uint32_t>((chunk & 7) ^ (r & 7)) << 4);
                    uint32_t v[4];
                    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at));
                    bool hit = false;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        constexpr uint32_t m = TcType<T>::kNonFinite;
                        if ((v[e] & m) == m) {
                            v[e] &= 0xFFFF0000u;
                            hit = true;
                        }
                        if ((v[e] & (m << 16)) == m << 16) {
                            v[e] &= 0x0000FFFFu;
                            hit = true;
                        }
                    }
                    if (hit) {
                        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
                        *reinterpret_cast<volatile int *>(&x.bad[check_seg & (kSlots - 1)]) = 1;
                    }
                }
            }
            fence_proxy_async();
            mbar_arrive(smem_addr(&x.full[told % NB]));
        }
    };
    // one more buffer may be issued; announces older ones first when it has to wait
    auto claim = [&]() {
        const uint32_t bar = smem_addr(&x.empty[next % NB]), parity = ((next / NB) & 1) ^ 1;
        if (!mbar_try(bar, parity)) {
            copy_wait<0>();
            announce(next);
            mbar_wait(bar, parity, abort);
        }
    };
    auto issued = [&]() {
        copy_commit();
        next++;
        if (next - told > 2) {
            copy_wait<2>();
            announce(next - 2);
        }
    };
    TreeWalk walk;
    walk.begin(x);
    int tile = 0;
    while (walk.next(a, units)) {
        const int h = walk.u / g.mtiles;
        const T *kh = static_cast<const T *>(a.k) + h * a.k_hs + chunk * 8, *vh = static_cast<const T *>(a.v) + h * a.v_hs + chunk * 8;
        for (int j = walk.j0; j < walk.j1; j++, tile++) {
            const int64_t pos = static_cast<int64_t>(j) * kTile + pw * 32 + lane;
            int slot = 0;
            const int64_t page = pos < walk.length ? tree_page(a, walk.b, pos, &slot) : -1;
            const unsigned ok = __ballot_sync(kFullMask, page >= 0);
            const int64_t k_at = page * a.k_ps + slot * a.k_ts, v_at = page * a.v_ps + slot * a.v_ts;
            claim();
            if (lane == 0)
                x.valid[tile & (kSlots - 1)][pw] = ok;
            uint32_t dst = ring + static_cast<uint32_t>(next % NB) * Shape::kBuffer + column + static_cast<uint32_t>(pw * 32 + sub) * 128;
#pragma unroll
            for (int i = 0; i < 32 / ROWS; i++) {
                const int r = sub + i * ROWS;
                const int64_t at = __shfl_sync(kFullMask, k_at, r);
                const bool good = ok >> r & 1u;
                copy16_or_zero(dst + static_cast<uint32_t>(i * ROWS) * 128 + (static_cast<uint32_t>((chunk & 7) ^ (r & 7)) << 4),
                               good ? static_cast<const void *>(kh + at) : a.q, good ? 16u : 0u);
            }
            issued();
            claim();
            dst = ring + static_cast<uint32_t>(next % NB) * Shape::kBuffer + column + static_cast<uint32_t>(pw * 32 + sub) * 128;
#pragma unroll
            for (int i = 0; i < 32 / ROWS; i++) {
                const int r = sub + i * ROWS;
                const int64_t at = __shfl_sync(kFullMask, v_at, r);
                const bool good = ok >> r & 1u;
                copy16_or_zero(dst + static_cast<uint32_t>(i * ROWS) * 128 + (static_cast<uint32_t>((chunk & 7) ^ (r & 7)) << 4),
                               good ? static_cast<const void *>(vh + at) : a.q, good ? 16u : 0u);
            }
            if (static_cast<int64_t>(j + 1) * kTile > walk.context) {
                if (check_buffer >= told) {  // an earlier one is still to be announced
                    copy_wait<0>();
                    announce(next);
                }
                check_buffer = next;
                check_from = walk.context - static_cast<int64_t>(j) * kTile - pw * 32;
                check_seg = walk.seg;
            }
            issued();
        }
    }
    copy_wait<0>();
    announce(next);
}

// ---- products ----
template <typename T, int D, int ROWT>
__device__ __forceinline__ void tree_product_role(const TreeMmaArgs &g, TreeMmaExtras &x, uint32_t q_smem, uint32_t ring, int units) {
    using Shape = TreeMmaShape<D, ROWT>;
    constexpr int NB = Shape::kRing;
    constexpr uint32_t qk = mma_instruction<T>(128, kTile, false), pv = mma_instruction<T>(128, D, true);
    volatile int *abort = &x.abort;
    const uint32_t tmem = x.tmem;
    int scores[2] = {0, 0};  // S tiles issued for a group
    int weights[2] = {0, 0}; // P tiles multiplied
    int first = 0;           // first buffer of the unit's tiles (keys, values, keys, ...)
    bool ok = true;
    auto wait_buffer = [&](int n) { ok = mbar_wait(smem_addr(&x.full[n % NB]), (n / NB) & 1, abort) && ok; };
    auto score = [&](int w, int n) {  // S_w = Q K^T from buffer n
        if (ok) {
            const uint32_t qb = q_smem + (ROWT == 2 ? static_cast<uint32_t>(w) * (128 * D * 2) : 0u), kb = ring + static_cast<uint32_t>(n % NB) * Shape::kBuffer;
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < D / 16; k++)
                mma_ss(tmem + w * kTile, mma_operand(qb + (k >> 2) * (128 * 128) + (k & 3) * 32, 16, 1024),
                       mma_operand(kb + (k >> 2) * (kTile * 128) + (k & 3) * 32, 16, 1024), qk, k > 0);
        }
        mma_commit(smem_addr(&x.s_ready[w]));
        scores[w]++;
    };
    auto weigh = [&](int w, int n, bool add) {  // O_w += P V from buffer n
        ok = mbar_wait(smem_addr(&x.p_ready[w]), weights[w] & 1, abort) && ok;
        if (ok) {
            const uint32_t vb = ring + static_cast<uint32_t>(n % NB) * Shape::kBuffer;
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < kTile / 16; k++)
                mma_ts(tmem + 2 * kTile + w * D, tmem + w * kTile + k * 8, mma_operand(vb + k * 2048, kTile * 128, 1024), pv, add || k > 0);
        }
        mma_commit(smem_addr(&x.pv_done[w]));
        weights[w]++;
    };
    // P lies where the next S goes: the product that reads it has to be done
    auto wait_weighed = [&](int w) { ok = mbar_wait(smem_addr(&x.pv_done[w]), (weights[w] - 1) & 1, abort) && ok; };
    auto release = [&](int n) { mma_commit(smem_addr(&x.empty[n % NB])); };
    TreeWalk walk;
    walk.begin(x);
    while (walk.next(g.a, units)) {
        const int n = walk.j1 - walk.j0;
        ok = mbar_wait(smem_addr(&x.q_ready), walk.seg & 1, abort) && ok;
        if (ROWT == 2) {
            wait_buffer(first);
            score(0, first);
            score(1, first);
            release(first);
            for (int t = 0; t < n; t++) {
                const int k_next = first + 2 * t + 2, v_now = first + 2 * t + 1;
                wait_buffer(v_now);
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    weigh(w, v_now, t > 0);
                    if (w == 1)
                        release(v_now);
                    if (t + 1 < n) {
                        if (w == 0)
                            wait_buffer(k_next);
                        wait_weighed(w);
                        score(w, k_next);
                        if (w == 1)
                            release(k_next);
                    }
                }
            }
        } else {
            for (int t = 0; t < 2 && t < n; t++) {
                wait_buffer(first + 2 * t);
                score(t, first + 2 * t);
                release(first + 2 * t);
            }
            for (int t = 0; t < n; t++) {
                const int w = t & 1, v_now = first + 2 * t + 1;
                wait_buffer(v_now);
                weigh(w, v_now, t > 1);
                release(v_now);
                if (t + 2 < n) {
                    wait_buffer(first + 2 * t + 4);
                    wait_weighed(w);
                    score(w, first + 2 * t + 4);
                    release(first + 2 * t + 4);
                }
            }
        }
        first += 2 * n;
    }
    // tensor memory may be given back once nothing writes to it any more
    for (int w = 0; w < 2; w++)
        if (weights[w] > 0)
            wait_weighed(w);
}

// ---- softmax and output ----
template <typename T, int D, int ROWT>
__device__ __forceinline__ void tree_softmax_role(const TreeMmaArgs &g, TreeMmaExtras &x, unsigned char *q_ptr, int units) {
    const TreeArgs &a = g.a;
    const int tid = threadIdx.x, w = tid >> 7, trow = tid & 127;
    volatile int *abort = &x.abort;
    const uint32_t lanes = static_cast<uint32_t>((tid >> 5) & 3) << 21;  // this warp's quarter of the tensor-memory lanes
    const uint32_t t_s = x.tmem + lanes + w * kTile, t_o = x.tmem + lanes + 2 * kTile + w * D;
    int seen = 0;  // tiles that this group has worked on
    int tile = 0;  // tiles of the units before this one
    bool ok = true;
    TreeWalk walk;
    walk.begin(x);
    while (walk.next(a, units)) {
        const int b = walk.b, h = walk.u / g.mtiles, n = walk.j1 - walk.j0;
        const int row = walk.u % g.mtiles * (ROWT * 128) + (ROWT == 2 ? w * 128 : 0) + trow;
        const bool row_ok = row < a.rows;
        const int node = row_ok ? row / a.group : 0, head = h * a.group + (row_ok ? row % a.group : 0);
        const bool live = row_ok && node < walk.used;
        const bool warp_live = __any_sync(kFullMask, live);
        const bool drafted = static_cast<int64_t>(walk.j1) * kTile > walk.context;
        if (drafted && trow < a.nodes) {
            const int up = a.parents ? a.parents[static_cast<int64_t>(b) * a.nodes + trow] : trow - 1;
            x.parents[w][trow] = up >= 0 && up < trow ? up : 255;
        }
        // both groups are done with the unit before: its queries (every S has been made) and its flags may go
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (tid == 0 && walk.seg > 0)
            x.bad[(walk.seg - 1) & (kSlots - 1)] = 0;
        {
            constexpr int PIECES = ROWT == 2 ? D / 8 : D / 16;
            const int from = ROWT == 2 ? 0 : w * PIECES;
            const T *src = static_cast<const T *>(a.q) + b * a.q_bs + node * a.q_ns + head * a.q_hs;
            unsigned char *dst = q_ptr + (ROWT == 2 ? w * (128 * D * 2) : 0) + trow * 128;
#pragma unroll
            for (int c = 0; c < PIECES; c++) {
                const int piece = from + c;
                uint4 v = live ? *reinterpret_cast<const uint4 *>(src + piece * 8) : make_uint4(0, 0, 0, 0);
                v.x = (v.x ^ g.flip) & g.mask, v.y = (v.y ^ g.flip) & g.mask, v.z = (v.z ^ g.flip) & g.mask, v.w = (v.w ^ g.flip) & g.mask;
                *reinterpret_cast<uint4 *>(dst + (piece >> 3) * (128 * 128) + (((piece & 7) ^ (trow & 7)) << 4)) = v;
            }
        }
        fence_proxy_async();
        mbar_arrive(smem_addr(&x.q_ready));
        uint32_t anc[kTreeWords] = {};
        if (drafted && live) {
            int at = node;
            while (true) {
#pragma unroll
                for (int e = 0; e < kTreeWords; e++)
                    anc[e] |= at >> 5 == e ? 1u << (at & 31) : 0u;
                const int up = x.parents[w][at];
                if (up == 255)
                    break;
                at = up;
            }
        }

        float m_ref = -INFINITY, l = 0.0f;  // reference of the exponents in log2 units, sum of the weights
        int mine = 0;
        for (int t = ROWT == 2 ? 0 : w; t < n; t += ROWT == 2 ? 1 : 2, mine++) {
            ok = __all_sync(kFullMask, mbar_wait(smem_addr(&x.s_ready[w]), seen & 1, abort)) && ok;
            seen++;
            if (warp_live && ok) {
                tc_fence_after();
                uint32_t s[4][32];
#pragma unroll
                for (int c = 0; c < 4; c++)
                    tmem_load32(t_s + 32 * c, s[c]);
                tmem_wait_load();
#pragma unroll
                for (int c = 0; c < 4; c++)
                    tmem_settle32(s[c]);
                const int64_t t0 = static_cast<int64_t>(walk.j0 + t) * kTile;
                const uint4 there = *reinterpret_cast<const uint4 *>(x.valid[(tile + t) & (kSlots - 1)]);
                if (t0 + kTile > walk.context || (there.x & there.y & there.z & there.w) != 0xFFFFFFFFu) {
                    const uint32_t valid[4] = {there.x, there.y, there.z, there.w};
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const int64_t j = t0 + 32 * c - walk.context;  // node at the first of these positions; negative: context
                        uint32_t see = 0;
                        if (j <= -32) {
                            see = 0xFFFFFFFFu;
                        } else if (j < kTreeMaxNodes) {
                            const int sh = static_cast<int>(j) & 31, word = static_cast<int>(j) >> 5;  // -1 .. 3
                            uint32_t lo = 0xFFFFFFFFu, hi = 0;
#pragma unroll
                            for (int e = 0; e < kTreeWords; e++) {
                                lo = word == e ? anc[e] : lo;
                                hi = word + 1 == e ? anc[e] : hi;
                            }
                            see = __funnelshift_r(lo, hi, sh);
                        }
                        see = live ? see & valid[c] : 0u;
#pragma unroll
                        for (int i = 0; i < 32; i++)
                            s[c][i] = see >> i & 1u ? s[c][i] : 0xFF800000u;
                    }
                }
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 32; i++)
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        top[c] = fmaxf(top[c], __uint_as_float(s[c][i]));
                const float m_tile = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * g.scale;
                if (__any_sync(kFullMask, m_tile > m_ref + kGrow)) {
                    // (also the first tile of a unit: m_ref = -inf, nothing to rescale yet)
                    const float m_new = fmaxf(m_ref, m_tile), keep = m_ref == m_new ? 1.0f : exp2_approx(m_ref - m_new);
                    m_ref = m_new;
                    l *= keep;
                    if (mine > 0) {
#pragma unroll
                        for (int c = 0; c < D / 32; c++) {
                            uint32_t o[32];
                            tmem_load32(t_o + 32 * c, o);
                            tmem_wait_load();
                            tmem_settle32(o);
#pragma unroll
                            for (int i = 0; i < 32; i++)
                                o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
                            tmem_store32(t_o + 32 * c, o);
                        }
                    }
                }
                const float off = (m_ref == -INFINITY ? 0.0f : m_ref) - kBias;
                float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    uint32_t p[32];
#pragma unroll
                    for (int i = 0; i < 32; i++) {
                        const int c = half * 2 + (i >> 4), e = (i & 15) * 2;
                        const float p0 = exp2_approx(fmaf(__uint_as_float(s[c][e]), g.scale, -off));
                        const float p1 = exp2_approx(fmaf(__uint_as_float(s[c][e + 1]), g.scale, -off));
                        sum[(i & 1) * 2] += p0;
                        sum[(i & 1) * 2 + 1] += p1;
                        p[i] = TcType<T>::pack(p0, p1);
                    }
                    tmem_store32(t_s + 32 * half, p);
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                tmem_wait_store();
            }
            tc_fence_before();
            mbar_arrive(smem_addr(&x.p_ready[w]));
        }
        if (mine > 0)
            ok = __all_sync(kFullMask, mbar_wait(smem_addr(&x.pv_done[w]), (seen - 1) & 1, abort)) && ok;
        __syncwarp();
        tc_fence_after();

        // ---- the unit's rows, or this CTA's part of them ----
        float m = m_ref == -INFINITY ? -INFINITY : m_ref - kBias;
        float f0 = 1.0f, f1 = 0.0f;
        constexpr int COLS = ROWT == 2 ? D : D / 2;  // a group's columns of the output
        if (ROWT == 1) {
            x.ml[w][trow] = make_float2(m, l);
            tc_fence_before();
            asm volatile("bar.sync 1, 256;" ::: "memory");
            tc_fence_after();
            const float2 u0 = x.ml[0][trow], u1 = x.ml[1][trow];
            m = fmaxf(u0.x, u1.x);
            const float base = m == -INFINITY ? 0.0f : m;
            f0 = exp2_approx(u0.x - base);
            f1 = exp2_approx(u1.x - base);
            l = u0.y * f0 + (n > 1 ? u1.y * f1 : 0.0f);
        }
        const bool whole = walk.whole();
        const int64_t slot = (static_cast<int64_t>(blockIdx.x) * 2 + (walk.seg > 0)) * (ROWT * 128) + (ROWT == 2 ? w * 128 : 0) + trow;
        T *o_row = static_cast<T *>(a.out) + b * a.o_bs + node * a.o_ns + head * a.o_hs;
        const bool empty = l == 0.0f;
        const float inv = empty ? 0.0f : 1.0f / l;
        const bool broken = *reinterpret_cast<volatile int *>(&x.bad[walk.seg & (kSlots - 1)]) != 0;
        if (__any_sync(kFullMask, row_ok)) {
#pragma unroll
            for (int c = 0; c < COLS / 32; c++) {
                const int col = (ROWT == 2 ? 0 : w * COLS) + 32 * c;
                uint32_t o[32];
                if (ROWT == 2) {
                    tmem_load32(t_o + col, o);
                    tmem_wait_load();
                    tmem_settle32(o);
                } else {
                    const uint32_t o0 = x.tmem + lanes + 2 * kTile + col;
                    tmem_load32(o0, o);
                    tmem_wait_load();
                    tmem_settle32(o);
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        o[i] = __float_as_uint(__uint_as_float(o[i]) * f0);
                    if (n > 1) {
                        uint32_t o2[32];
                        tmem_load32(o0 + D, o2);
                        tmem_wait_load();
                        tmem_settle32(o2);
#pragma unroll
                        for (int i = 0; i < 32; i++)
                            o[i] = __float_as_uint(fmaf(__uint_as_float(o2[i]), f1, __uint_as_float(o[i])));
                    }
                }
                if (row_ok) {
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        o[i] = empty ? 0u : o[i];
                    if (broken && live) {  // values that are not finite: a positive weight of them is the value itself
                        for (int64_t pos = max(walk.context, static_cast<int64_t>(walk.j0) * kTile);
                             pos < min(walk.length, static_cast<int64_t>(walk.j1) * kTile); pos++) {
                            const int j = static_cast<int>(pos - walk.context);
                            int at = 0;
                            const int64_t page = tree_page(a, b, pos, &at);
                            uint32_t word = 0;
#pragma unroll
                            for (int e = 0; e < kTreeWords; e++)
                                word = j >> 5 == e ? anc[e] : word;
                            if (page < 0 || !(word >> (j & 31) & 1u))
                                continue;
                            const T *v = static_cast<const T *>(a.v) + page * a.v_ps + at * a.v_ts + h * a.v_hs + col;
#pragma unroll
                            for (int i = 0; i < 32; i++) {
                                const float f = Elem<T>::from_storage(v[i]);
                                if (!(fabsf(f) < INFINITY))
                                    o[i] = __float_as_uint(__uint_as_float(o[i]) + f);
                            }
                        }
                    }
                    if (!ok) {  // a wait ran out: the result shows it
#pragma unroll
                        for (int i = 0; i < 32; i++)
                            o[i] = 0x7FC00000u;
                    }
                    if (whole) {
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            uint32_t v[4];
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const float lo = __uint_as_float(o[i + 2 * e]), hi = __uint_as_float(o[i + 2 * e + 1]);
                                v[e] = TcType<T>::pack(empty ? lo : lo * inv, empty ? hi : hi * inv);
                            }
                            *reinterpret_cast<uint4 *>(o_row + col + i) = make_uint4(v[0], v[1], v[2], v[3]);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            *reinterpret_cast<uint4 *>(a.part_o + slot * D + col + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    }
                }
                __syncwarp();
            }
            if (row_ok && (ROWT == 2 || w == 0)) {
                if (!whole)
                    a.part_ml[slot] = make_float2(m, l);
                else if (a.lse)
                    a.lse[(static_cast<int64_t>(b) * a.nodes + node) * a.q_heads + head] = empty ? -INFINITY : (m + log2f(l)) * kLn2;
            }
        }
        tile += n;
        tc_fence_before();  // the next unit's products may overwrite what was read
    }
}

template <typename T, int D, int ROWT>
__global__ void __launch_bounds__(kMmaThreads, 1) tree_attention_mma_kernel(const TreeMmaArgs g) {
    using Shape = TreeMmaShape<D, ROWT>;
    extern __shared__ __align__(1024) unsigned char smem[];
    TreeMmaExtras &x = *reinterpret_cast<TreeMmaExtras *>(smem + Shape::kQ + Shape::kRing * Shape::kBuffer);
    const TreeArgs &a = g.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int units = a.kv_heads * g.mtiles;

    // this CTA's range of the list of all tiles
    int64_t *s_scan = reinterpret_cast<int64_t *>(smem);
    const int per = (a.batch + kMmaThreads - 1) / kMmaThreads;
    const int b0 = min(a.batch, tid * per), b1 = min(a.batch, b0 + per);
    int64_t sum = 0;
    for (int b = b0; b < b1; b++)
        sum += static_cast<int64_t>(tree_tiles(a, b)) * units;
    int64_t upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(kFullMask, upto, o);
        upto += lane >= o ? v : 0;
    }
    if (lane == 31)
        s_scan[warp] = upto;
    if (tid == 0) {
        for (int i = 0; i < 8; i++) {
            mbar_init(smem_addr(&x.full[i]), 128);
            mbar_init(smem_addr(&x.empty[i]), 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(smem_addr(&x.s_ready[i]), 1);
            mbar_init(smem_addr(&x.p_ready[i]), 128);
            mbar_init(smem_addr(&x.pv_done[i]), 1);
        }
        mbar_init(smem_addr(&x.q_ready), 256);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        x.abort = 0;
        x.left = 0;
        for (int i = 0; i < kSlots; i++)
            x.bad[i] = 0;
    }
    __syncthreads();
    int64_t total = 0, before = upto - sum;
    for (int i = 0; i < kMmaThreads / 32; i++) {
        before += i < warp ? s_scan[i] : 0;
        total += s_scan[i];
    }
    const int64_t lo = blockIdx.x * total / gridDim.x, hi = (blockIdx.x + 1) * total / gridDim.x;
    if (blockIdx.x == 0) {
        int64_t at = before;
        for (int b = b0; b < b1; b++) {
            g.starts[b] = at;
            at += static_cast<int64_t>(tree_tiles(a, b)) * units;
        }
        if (tid == 0)
            g.starts[a.batch] = total;
    }
    if (lo < hi && lo >= before && lo < before + sum) {
        int64_t at = before;
        int b = b0, tiles = tree_tiles(a, b);
        while (lo >= at + static_cast<int64_t>(tiles) * units) {
            at += static_cast<int64_t>(tiles) * units;
            tiles = tree_tiles(a, ++b);
        }
        x.begin_b = b;
        x.begin_u = static_cast<int>((lo - at) / tiles);
        x.begin_j = static_cast<int>((lo - at) % tiles);
        x.left = hi - lo;
    }
    if (lo >= hi)
        return;  // fewer tiles than CTAs
    if (warp == 12)
        tmem_alloc(smem_addr(&x.tmem), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t q_smem = smem_addr(smem), ring = q_smem + Shape::kQ;

    // registers: 128 a thread at launch, 2 x 184 + 88 + 56 = 4 x 128
    if (warp < 8) {
        set_registers_up<184>();
        tree_softmax_role<T, D, ROWT>(g, x, smem, units);
    } else if (warp < 12) {
        set_registers_down<88>();
        tree_copy_role<T, D, ROWT>(g, x, ring, units);
    } else {
        set_registers_down<56>();
        if (warp == 12) {
            if (lane == 0)
                tree_product_role<T, D, ROWT>(g, x, q_smem, ring, units);
            __syncwarp();
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 12)
        tmem_free(x.tmem, 512);
}

// ---- join: one warp a row of a unit that several CTAs worked on ----
constexpr int kMmaJoinWarps = 8;

template <typename T, int D, int ROWT>
__global__ void __launch_bounds__(kMmaJoinWarps * 32) tree_attention_mma_join_kernel(const TreeMmaArgs g, int ctas) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const TreeArgs &a = g.a;
    const int lane = threadIdx.x & 31, units = a.kv_heads * g.mtiles;
    const int b = blockIdx.x / units, u = blockIdx.x % units;
    const int in_unit = blockIdx.y * kMmaJoinWarps + (threadIdx.x >> 5), row = u % g.mtiles * (ROWT * 128) + in_unit;
    if (row >= a.rows)
        return;
    const int64_t total = g.starts[a.batch], first = g.starts[b], tiles = (g.starts[b + 1] - first) / units;
    const int64_t lo = first + u * tiles, hi = lo + tiles;
    const int c0 = static_cast<int>(((lo + 1) * ctas - 1) / total), c1 = static_cast<int>((hi * ctas - 1) / total);
    if (c0 == c1)
        return;  // written out by the one CTA
    // CTA c's part lies in its first slot when its range begins inside the unit, else in its second; a range may be empty
    auto part = [&](int c) -> int64_t {
        const int64_t from = c * total / ctas;
        if (from == (c + 1) * total / ctas)
            return -1;
        return (static_cast<int64_t>(c) * 2 + (from < lo)) * (ROWT * 128) + in_unit;
    };
    float top = -INFINITY;
    for (int c = c0 + lane; c <= c1; c += 32)
        if (const int64_t i = part(c); i >= 0)
            top = fmaxf(top, a.part_ml[i].x);
    top = warp_max(top);
    const float base = top == -INFINITY ? 0.0f : top;
    float l = 0.0f, acc[D / 32];
#pragma unroll
    for (int e = 0; e < D / 32; e++)
        acc[e] = 0.0f;
#pragma unroll 4
    for (int c = c0; c <= c1; c++) {
        const int64_t i = part(c);
        if (i < 0)
            continue;
        const float2 ml = a.part_ml[i];
        const float f = exp2f(ml.x - base);
        l = fmaf(f, ml.y, l);
#pragma unroll
        for (int e = 0; e < D / 32; e++)
            acc[e] = fmaf(f, a.part_o[i * D + lane + 32 * e], acc[e]);
    }
    const int node = row / a.group, head = u / g.mtiles * a.group + row % a.group;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T *o = static_cast<T *>(a.out) + b * a.o_bs + node * a.o_ns + head * a.o_hs;
#pragma unroll
    for (int e = 0; e < D / 32; e++)
        o[lane + 32 * e] = Elem<T>::to_storage(l == 0.0f ? 0.0f : acc[e] * inv);
    if (a.lse && lane == 0)
        a.lse[(static_cast<int64_t>(b) * a.nodes + node) * a.q_heads + head] = l == 0.0f ? -INFINITY : (top + log2f(l)) * kLn2;
}

// ---- host side ----
bool tree_mma_serves(const vkop_tree_attention_desc &d) {
    return d.dtype != VKOP_F32 && (d.head_dim == 64 || d.head_dim == 128);
}

static int64_t slot_rows(const TreeArgs &a) { return a.rows > 128 ? 256 : 128; }

size_t tree_mma_workspace(const vkop_tree_attention_desc &d) {
    const int64_t rows = static_cast<int64_t>(d.nodes) * (d.q_heads / d.kv_heads) > 128 ? 256 : 128;
    const size_t starts = (static_cast<size_t>(d.batch + 1) * 8 + 15) / 16 * 16;
    return starts + static_cast<size_t>(kMmaCtas) * 2 * rows * (d.head_dim + 2) * sizeof(float);
}

template <typename T, int D, int ROWT>
static int launch_mma_t(const TreeMmaArgs &g, cudaStream_t stream) {
    constexpr int smem = TreeMmaShape<D, ROWT>::kSmem;
    if (cudaFuncSetAttribute(tree_attention_mma_kernel<T, D, ROWT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
        cudaGetLastError();
        return VKOP_CUDA_ERROR;
    }
    tree_attention_mma_kernel<T, D, ROWT><<<kMmaCtas, kMmaThreads, smem, stream>>>(g);
    note_launch();
    if (check_launch() != VKOP_OK)
        return VKOP_CUDA_ERROR;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(g.a.batch * g.a.kv_heads * g.mtiles),
                       static_cast<unsigned>((min(g.a.rows, ROWT * 128) + kMmaJoinWarps - 1) / kMmaJoinWarps));
    cfg.blockDim = dim3(kMmaJoinWarps * 32);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, tree_attention_mma_join_kernel<T, D, ROWT>, g, kMmaCtas) != cudaSuccess) {
        cudaGetLastError();
        return VKOP_CUDA_ERROR;
    }
    note_launch();
    return VKOP_OK;
}

template <typename T>
static int launch_mma_type(const TreeMmaArgs &g, cudaStream_t stream) {
    if (g.a.head_dim == 64)
        return g.a.rows > 128 ? launch_mma_t<T, 64, 2>(g, stream) : launch_mma_t<T, 64, 1>(g, stream);
    return g.a.rows > 128 ? launch_mma_t<T, 128, 2>(g, stream) : launch_mma_t<T, 128, 1>(g, stream);
}

int launch_tree_mma(const TreeArgs &args, int dtype, void *workspace, cudaStream_t stream) {
    TreeMmaArgs g;
    g.a = args;
    g.starts = static_cast<int64_t *>(workspace);
    const size_t starts = (static_cast<size_t>(args.batch + 1) * 8 + 15) / 16 * 16;
    g.a.part_ml = reinterpret_cast<float2 *>(static_cast<char *>(workspace) + starts);
    g.a.part_o = reinterpret_cast<float *>(g.a.part_ml + kMmaCtas * 2 * slot_rows(args));
    g.mtiles = args.rows > 128 ? (args.rows + 255) / 256 : 1;
    g.scale = args.scale_log2 == 0.0f ? 1.0f : fabsf(args.scale_log2);
    g.mask = args.scale_log2 == 0.0f ? 0u : 0xFFFFFFFFu;
    g.flip = args.scale_log2 < 0.0f ? 0x80008000u : 0u;
    return dtype == VKOP_F16 ? launch_mma_type<__half>(g, stream) : launch_mma_type<__nv_bfloat16>(g, stream);
}

}  // namespace vkop_cuda
