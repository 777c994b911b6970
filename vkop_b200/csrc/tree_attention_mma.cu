// Attention of a tree of drafted tokens over a paged cache on the tensor cores: 16-bit types, head sizes 64 and 128.
//
// The rows that share a cache head (nodes x query heads a cache head) fill the M dimension of 128-row products; 64 or 128
// cached positions are the N dimension of S = Q K^T, 64 the K dimension of O += P V.  Roles of a CTA (one a SM, 16 warps):
//   warps 0-7    softmax: two groups of 128 threads, a thread a row.  With more than 128 rows each group has its own 128 and
//                both see every position (ROWT = 2); otherwise one group takes the first, the other the second half of every
//                tile of 128 positions and their sums are joined at the end (ROWT = 1).
//   warps 8-11   copies: a tile's keys and values come from their pages into a ring of buffers, in rows of 128 bytes with the
//                128-byte swizzle that the products read.  Where 32 rows in turn are all there and belong to the context,
//                and the page size is a multiple of 8, tensor-map copies of 8 to 32 rows bring them; the others (the end of
//                a sequence, missing pages, other page sizes) are gathered by 16-byte copies, which leave zeros where
//                nothing is.
//   warp 14      products, for the groups in turn.  S (then P in its place) and O live in tensor memory.  ROWT = 1: two S
//                tiles of 64 positions a group alternate, so that one is being made while the other is turned into weights.
//                ROWT = 2: one S tile of 128 positions a group, the groups take turns (products 128 wide need a quarter less
//                of the tensor pipe, which reads 128 bytes a clock of operands from shared memory).  The products of a warp
//                are carried out in the order of their issue: the S that overwrites a P is issued behind the product that
//                reads it, without a wait in between.
//
// S: exponents are taken relative to a reference that follows the row's maximum only when it grows by more than 2^8 (the sums
// are rescaled then, in tensor memory); P is scaled by 2^kBias so that 16-bit weights stay clear of the subnormal range.
//
// Work is cut without regard to sequence borders: all tiles of the call, sequence by sequence, head by head, are one list that
// the CTAs share out evenly, whatever the lengths of the sequences.  A (sequence, head, rows) unit that one CTA holds entirely
// is written out; of others every CTA leaves its part in its own two slots of the scratch memory (first and last unit of its
// range) and the join adds them up.  Where sequences are short, whole units are shared out instead: no scan, no
// parts, no second launch (whole_units below).
//
// Bound: reading the cache once from HBM for few rows a head; around 256 rows the products and the exponentials
// (16 a clock and SM) take as long as the copies.
#include <cuda.h>

#include <atomic>

#include "tensor_core.cuh"
#include "tree_attention.cuh"

namespace vkop_cuda {

constexpr int kMmaThreads = 512;
constexpr int kTile = 128;       // positions a tile: what a buffer of the ring holds
constexpr int kHalf = 64;        // positions a product
constexpr int kMmaCtas = 148;
constexpr int kProductWarp = 14;  // not on the scheduler of warps 0 and 4, which have all the rows where they are few
constexpr float kBias = 6.0f;    // log2 of the scale of the weights
constexpr float kGrow = 8.0f;    // log2 of the growth of the maximum that is let pass; 2^(6 + 8) < 65504
constexpr int kSlots = 8;        // tiles (and units) whose flags may be alive at once: more than a ring holds

struct TreeMmaArgs {
    TreeArgs a;
    int box_rows;     // rows of a tensor-map copy; 0: rows are gathered one by one
    int page_shift;   // log2(page_size), -1 where it is not a power of two
    int64_t *starts;  // [batch + 1] first place of a sequence in the list
    int whole;        // whole units are shared out
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
    static constexpr int kExtras = 3 * 1024;
    static constexpr int kUnitCost = 3;  // what a change of units costs, in tiles
    static constexpr int kSmem = kQ + kRing * kBuffer + kExtras;
};

struct TreeMmaExtras {
    uint64_t full[8], empty[8], s_ready[2][2], p_ready[2][2], pv_done[2][2], q_ready, done;
    int64_t left;
    uint32_t tmem;
    int abort, begin_b, begin_u, begin_j, units_left;
    alignas(16) uint32_t valid[kSlots][4];
    int bad[kSlots];
    uint8_t parents[2][kTreeMaxNodes];
    float2 ml[2][128];
};
static_assert(sizeof(TreeMmaExtras) <= 3 * 1024, "extras");

__device__ __forceinline__ int tree_tiles(const TreeArgs &a, int b) {
    const int64_t length = tree_length(a, b);
    return length <= 0 ? 1 : static_cast<int>((length + kTile - 1) / kTile);
}

// The units that a CTA's range of the list runs through.  Every unit is as long as its tiles and COST places that stand for
// the work of changing units.
template <int COST>
struct TreeWalk {
    int64_t left;  // places still to come
    int b, u, j0, j1, tiles, seg, units_left;
    bool first;  // the range begins inside this unit (its part goes to the CTA's first slot)
    int64_t context, length;
    int used;
    __device__ __forceinline__ void begin(const TreeMmaExtras &x) {
        left = x.left;
        b = x.begin_b;
        u = x.begin_u;
        j1 = x.begin_j;
        units_left = x.units_left;
        seg = -1;
        tiles = -1;
        first = true;
    }
    __device__ __forceinline__ bool next(const TreeArgs &a, int units) {
        while (left > 0 && units_left != 0) {
            if (tiles < 0) {
                context = tree_context(a, b);
                used = tree_used(a, b);
                length = tree_length(a, b);
                tiles = length <= 0 ? 1 : static_cast<int>((length + kTile - 1) / kTile);
            }
            if (j1 < tiles) {
                if (seg >= 0)
                    first = false;
                j0 = j1;
                j1 = left < tiles - j0 ? j0 + static_cast<int>(left) : tiles;
                left -= j1 - j0;
                units_left--;
                seg++;
                return true;
            }
            left -= tiles + COST - j1;  // the places behind the tiles
            first = false;
            j1 = 0;
            if (++u == units) {
                u = 0;
                b++;
                tiles = -1;
            }
        }
        return false;
    }
    __device__ __forceinline__ bool whole() const { return j0 == 0 && j1 == tiles; }
};

// ---- copies ----
template <typename T, int D, int ROWT>
__device__ __forceinline__ void tree_copy_role(const TreeMmaArgs &g, const CUtensorMap *k_map, const CUtensorMap *v_map, TreeMmaExtras &x,
                                               uint32_t ring, int units) {
    using Shape = TreeMmaShape<D, ROWT>;
    constexpr int NB = Shape::kRing;
    constexpr int CHUNKS = D / 8;          // 16-byte pieces of a row
    constexpr int ROWS = 32 / CHUNKS;      // rows a warp gathers at a time
    const TreeArgs &a = g.a;
    const int lane = threadIdx.x & 31, pw = (threadIdx.x >> 5) & 3;
    const int chunk = lane % CHUNKS, sub = lane / CHUNKS;
    const uint32_t column = static_cast<uint32_t>(chunk >> 3) * (kTile * 128);
    volatile int *abort = &x.abort;
    int next = 0;  // buffers issued so far; this warp brings rows 32 pw .. 32 pw + 31 of each
    int told = 0;  // buffers announced so far; gathered ones follow when their copies have landed
    uint32_t boxed = 0;  // ring places whose buffer announces itself
    // a value tile with drafted rows: their values that are not finite are taken out (the epilogue adds them to the rows that
    // attend them; as a factor of a zero weight they would spoil the others)
    int check_from = 0, check_to = 0;  // drafted rows of the buffer in question, in rows of this warp
    int check_buffer = -1, check_seg = 0;
    auto announce = [&](int upto) {
        for (; told < upto; told++) {
            const int place = told % NB;
            if (boxed >> place & 1u) {
                boxed &= ~(1u << place);
                continue;
            }
            const uint32_t buf = ring + static_cast<uint32_t>(place) * Shape::kBuffer;
            if (told == check_buffer) {
#pragma unroll 1
                for (int r = sub + (max(check_from - sub, 0) + ROWS - 1) / ROWS * ROWS; r < check_to; r += ROWS) {
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
            __syncwarp();
            if (lane == 0)
                mbar_arrive(smem_addr(&x.full[place]));
        }
    };
    // the next buffer may be filled; older ones are announced first when that has to be waited for
    auto claim = [&]() {
        const uint32_t bar = smem_addr(&x.empty[next % NB]), parity = ((next / NB) & 1) ^ 1;
        if (!__all_sync(kFullMask, mbar_try(bar, parity))) {
            copy_wait<0>();
            announce(next);
            mbar_wait(bar, parity, abort);
            __syncwarp();
        }
    };
    auto issued = [&]() {  // a buffer is a group of copies, a self-announcing one an empty group
        copy_commit();
        next++;
        if (next - told > 2) {
            copy_wait<2>();
            announce(next - 2);
        }
    };
    // 32 rows by tensor-map copies
    auto boxes = [&](const CUtensorMap *map, int h, int page, int slot) {
        const uint32_t bar = smem_addr(&x.full[next % NB]), buf = ring + static_cast<uint32_t>(next % NB) * Shape::kBuffer;
        if (lane == 0)
            mbar_arrive_expect(bar, 32 * D * 2);
        const int row = lane / (D / 64) * g.box_rows;  // this lane's copy: rows from here on, one of the 64-wide column blocks
        const int page_of = __shfl_sync(kFullMask, page, row & 31), slot_of = __shfl_sync(kFullMask, slot, row & 31);
        if (row < 32)
            copy_box(buf + static_cast<uint32_t>(lane % (D / 64)) * (kTile * 128) + static_cast<uint32_t>(pw * 32 + row) * 128, map,
                     lane % (D / 64) * 64, slot_of, h, page_of, bar);
        boxed |= 1u << (next % NB);
        issued();
    };
    // 32 rows piece by piece, zeros where `ok` has no bit
    auto gather = [&](const T *head, int64_t at, unsigned ok) {
        const uint32_t dst = ring + static_cast<uint32_t>(next % NB) * Shape::kBuffer + column + static_cast<uint32_t>(pw * 32 + sub) * 128;
#pragma unroll
        for (int i = 0; i < 32 / ROWS; i++) {
            const int r = sub + i * ROWS;
            const int64_t from = __shfl_sync(kFullMask, at, r);
            const bool good = ok >> r & 1u;
            copy16_or_zero(dst + static_cast<uint32_t>(i * ROWS) * 128 + (static_cast<uint32_t>((chunk & 7) ^ (r & 7)) << 4),
                           good ? static_cast<const void *>(head + from) : a.q, good ? 16u : 0u);
        }
        issued();
    };
    TreeWalk<Shape::kUnitCost> walk;
    walk.begin(x);
    int tile = 0;
    while (walk.next(a, units)) {
        const int h = walk.u / g.mtiles;
        const T *kh = static_cast<const T *>(a.k) + h * a.k_hs + chunk * 8, *vh = static_cast<const T *>(a.v) + h * a.v_hs + chunk * 8;
        // this lane's row of a tile: its page (-1: none) and slot; looked up a tile ahead
        auto look = [&](int j, int *slot) {
            const uint32_t pos = static_cast<uint32_t>(j) * kTile + pw * 32 + lane;
            const uint32_t page = g.page_shift >= 0 ? pos >> g.page_shift : pos / static_cast<uint32_t>(a.page_size);
            *slot = static_cast<int>(pos - page * static_cast<uint32_t>(a.page_size));
            return j < walk.j1 && pos < walk.length && page < static_cast<uint32_t>(a.max_pages) ? a.table[walk.b * a.table_stride + page] : -1;
        };
        int slot, slot_next = 0, page_next = look(walk.j0, &slot_next);
        if (walk.seg == 0)
            asm volatile("bar.sync 2, 384;" ::: "memory");
        for (int j = walk.j0; j < walk.j1; j++, tile++) {
            const int page = page_next;
            slot = slot_next;
            page_next = look(j + 1, &slot_next);
            const unsigned ok = __ballot_sync(kFullMask, page >= 0 && page < a.num_pages);
            const int64_t drafted = walk.context - (static_cast<int64_t>(j) * kTile + pw * 32);  // first drafted row of the 32
            const bool whole = g.box_rows > 0 && ok == kFullMask && drafted >= 32;
            claim();
            if (lane == 0)
                x.valid[tile & (kSlots - 1)][pw] = ok;
            if (whole)
                boxes(k_map, h, page, slot);
            else
                gather(kh, page * a.k_ps + slot * a.k_ts, ok);
            claim();
            if (whole) {
                boxes(v_map, h, page, slot);
            } else {
                if (drafted < 32) {
                    if (check_buffer >= told) {  // an earlier one is still to be announced
                        copy_wait<0>();
                        announce(next);
                    }
                    check_buffer = next;
                    const int64_t rows = walk.length - (static_cast<int64_t>(j) * kTile + pw * 32);
                    check_from = static_cast<int>(drafted < 0 ? 0 : drafted);
                    check_to = static_cast<int>(rows < 0 ? 0 : rows < 32 ? rows : 32);
                    check_seg = walk.seg;
                }
                gather(vh, page * a.v_ps + slot * a.v_ts, ok);
            }
        }
    }
    copy_wait<0>();
    announce(next);
    // nothing of this CTA is in flight when it ends, not even after a wait that ran out (bounded as well)
    volatile int gave_up = 0;
    for (int n = next > NB ? next - NB : 0; n < next; n++)
        mbar_wait(smem_addr(&x.full[n % NB]), (n / NB) & 1, &gave_up);
}

// ---- products ----
template <typename T, int D, int ROWT>
__device__ __forceinline__ void tree_product_role(const TreeMmaArgs &g, TreeMmaExtras &x, uint32_t q_smem, uint32_t ring, int units) {
    using Shape = TreeMmaShape<D, ROWT>;
    constexpr int NB = Shape::kRing;
    constexpr uint32_t qk = mma_instruction<T>(128, ROWT == 2 ? kTile : kHalf, false), pv = mma_instruction<T>(128, D, true);
    volatile int *abort = &x.abort;
    const uint32_t tmem = __shfl_sync(kFullMask, x.tmem, 0);
    const uint32_t full = smem_addr(x.full), empty = smem_addr(x.empty), s_ready = smem_addr(x.s_ready), p_ready = smem_addr(x.p_ready),
                   pv_done = smem_addr(x.pv_done);
    // the path from the weights to the next S is what the softmax waits for: little is computed on it
    const uint64_t q_desc = mma_operand(q_smem, 16, 1024), k_desc = mma_operand(ring, 16, 1024), v_desc = mma_operand(ring, kTile * 128, 1024);
    int step = 0;  // S tiles made for each group
    uint32_t kn = 0, k_phase = 0, vn = 1, v_phase = 0;  // ring places of the keys and values to be used next, and their phases
    bool ok = true;
    auto wait = [&](uint32_t bar, uint32_t parity) {
        if (!mbar_try(bar, parity))
            ok = mbar_wait(bar, parity, abort) && ok;
    };
    auto advance = [&](uint32_t &n, uint32_t &phase) {  // keys and values alternate in the ring
        n += 2;
        if (n >= NB) {
            n -= NB;
            phase ^= 1;
        }
    };
    TreeWalk<Shape::kUnitCost> walk;
    walk.begin(x);
    while (walk.next(g.a, units)) {
        const int n = walk.j1 - walk.j0;
        wait(smem_addr(&x.q_ready), walk.seg & 1);
        if constexpr (ROWT == 2) {
            // tile i of a group: O += P V for its first half, then for its second and S(i + 1) in their place; -1 makes the first S
            for (int i = -1; i < n; i++, step++) {
                const bool weigh = i >= 0, make = i + 1 < n;
                const uint32_t phase = static_cast<uint32_t>(step - 1) & 1;
                if (make)
                    wait(full + kn * 8, k_phase);
                if (weigh)
                    wait(full + vn * 8, v_phase);
                const uint64_t kd = k_desc + (kn * Shape::kBuffer >> 4), vd = v_desc + (vn * Shape::kBuffer >> 4);
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    const uint32_t at = tmem + w * 2 * kHalf, to = tmem + 4 * kHalf + w * D;
                    if (weigh) {
                        wait(p_ready + w * 16, phase);
                        __syncwarp();
                        tc_fence_after();
                        if (elect_one() && ok) {
#pragma unroll
                            for (int k = 0; k < kHalf / 16; k++)
                                mma_ts(to, at + k * 8, vd + k * (2048 / 16), pv, i > 0 || k > 0);
                        }
                        __syncwarp();
                        wait(p_ready + w * 16 + 8, phase);
                    }
                    __syncwarp();
                    tc_fence_after();
                    if (elect_one()) {
                        if (weigh) {
                            if (ok) {
#pragma unroll
                                for (int k = 0; k < kHalf / 16; k++)
                                    mma_ts(to, at + kHalf + k * 8, vd + (kHalf * 128 + k * 2048) / 16, pv, true);
                            }
                            mma_commit(pv_done + w * 16);
                            if (w == 1)
                                mma_commit(empty + vn * 8);
                        }
                        if (make) {
                            if (ok) {
                                const uint64_t qd = q_desc + w * (128 * D * 2 / 16);
#pragma unroll
                                for (int k = 0; k < D / 16; k++)
                                    mma_ss(at, qd + ((k >> 2) * (128 * 128) + (k & 3) * 32) / 16, kd + ((k >> 2) * (kTile * 128) + (k & 3) * 32) / 16, qk, k > 0);
                            }
                            mma_commit(s_ready + w * 16);
                            if (w == 1)
                                mma_commit(empty + kn * 8);
                        }
                    }
                    __syncwarp();
                }
                if (make)
                    advance(kn, k_phase);
                if (weigh)
                    advance(vn, v_phase);
            }
            step--;
        } else {
            // step i of a group: O += P(i) V, then S(i + 2) in P(i)'s place; steps -2 and -1 make the first two S
            for (int i = -2; i < n; i++, step++) {
                const bool weigh = i >= 0, make = i + 2 < n;
                if (make)
                    wait(full + kn * 8, k_phase);
                if (weigh)
                    wait(full + vn * 8, v_phase);
                // P(i) and S(i + 2) have the same parity; tiles are counted over all units
                const uint32_t odd = static_cast<uint32_t>(step) & 1, phase = static_cast<uint32_t>(step - 2) >> 1 & 1;
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    const uint64_t kd = k_desc + ((kn * Shape::kBuffer + w * kHalf * 128) >> 4), vd = v_desc + ((vn * Shape::kBuffer + w * kHalf * 128) >> 4);
                    const uint32_t at = tmem + w * 2 * kHalf + odd * kHalf;
                    if (weigh)
                        wait(p_ready + w * 16 + odd * 8, phase);
                    __syncwarp();
                    tc_fence_after();
                    if (elect_one()) {
                        if (weigh) {
                            if (ok) {
#pragma unroll
                                for (int k = 0; k < kHalf / 16; k++)
                                    mma_ts(tmem + 4 * kHalf + w * D, at + k * 8, vd + k * (2048 / 16), pv, i > 0 || k > 0);
                            }
                            mma_commit(pv_done + w * 16 + odd * 8);
                            if (w == 1)
                                mma_commit(empty + vn * 8);
                        }
                        if (make) {
                            if (ok) {
#pragma unroll
                                for (int k = 0; k < D / 16; k++)
                                    mma_ss(at, q_desc + ((k >> 2) * (128 * 128) + (k & 3) * 32) / 16, kd + ((k >> 2) * (kTile * 128) + (k & 3) * 32) / 16, qk, k > 0);
                            }
                            mma_commit(s_ready + w * 16 + odd * 8);
                            if (w == 1)
                                mma_commit(empty + kn * 8);
                        }
                    }
                    __syncwarp();
                }
                if (make)
                    advance(kn, k_phase);
                if (weigh)
                    advance(vn, v_phase);
            }
            step -= 2;
        }
    }
    // tensor memory may be given back once nothing writes to it any more
    if (elect_one())
        mma_commit(smem_addr(&x.done));
    __syncwarp();
    volatile int gave_up = 0;
    mbar_wait(smem_addr(&x.done), 0, &gave_up);
}

// ---- softmax and output ----
template <typename T, int D, int ROWT>
__device__ __forceinline__ void tree_softmax_role(const TreeMmaArgs &g, TreeMmaExtras &x, unsigned char *q_ptr, int units) {
    using Shape = TreeMmaShape<D, ROWT>;
    const TreeArgs &a = g.a;
    const int tid = threadIdx.x, w = tid >> 7, trow = tid & 127;
    volatile int *abort = &x.abort;
    const uint32_t lanes = static_cast<uint32_t>((tid >> 5) & 3) << 21;  // this warp's quarter of the tensor-memory lanes
    const uint32_t s_base = x.tmem + lanes + w * 2 * kHalf, t_o = x.tmem + lanes + 4 * kHalf + w * D;
    int seen = 0;  // S tiles that this group has worked on
    int tile = 0;  // tiles of the units before this one
    bool ok = true;
    auto wait = [&](uint64_t &bar, int phase) {
        if (!__all_sync(kFullMask, mbar_try(smem_addr(&bar), phase & 1)))
            ok = __all_sync(kFullMask, mbar_wait(smem_addr(&bar), phase & 1, abort)) && ok;
    };
    // ROWT == 1: a barrier serves every other product (two may be under way): its parity tells a phase from its neighbours
    auto wait_weighed = [&](int k) { wait(x.pv_done[w][ROWT == 2 ? 0 : k & 1], ROWT == 2 ? k : k >> 1); };
    auto row_of = [&](const TreeWalk<Shape::kUnitCost> &at) { return at.u % g.mtiles * (ROWT * 128) + (ROWT == 2 ? w * 128 : 0) + trow; };
    // queries and parents of a unit into shared memory
    auto load_unit = [&](const TreeWalk<Shape::kUnitCost> &at, bool first) {
        if (static_cast<int64_t>(at.j1) * kTile > at.context && trow < a.nodes) {
            const int up = a.parents ? a.parents[static_cast<int64_t>(at.b) * a.nodes + trow] : trow - 1;
            x.parents[w][trow] = up >= 0 && up < trow ? up : 255;
        }
        // a warp loads whole rows, two (four) at a time, all loads before the stores
        constexpr int PIECES = D / 8, TOGETHER = 32 / PIECES, ROWS = ROWT == 2 ? 32 : 16, LOADS = ROWS / TOGETHER;
        const int lane = tid & 31, piece = lane % PIECES, r0 = (tid >> 5) * ROWS + lane / PIECES;
        const int base = at.u % g.mtiles * (ROWT * 128), h = at.u / g.mtiles;
        uint4 q[LOADS];
#pragma unroll
        for (int c = 0; c < LOADS; c++) {
            const int row = base + r0 + c * TOGETHER, node = row / a.group;
            q[c] = make_uint4(0, 0, 0, 0);
            if (row < a.rows && node < at.used)
                q[c] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + at.b * a.q_bs + node * a.q_ns + (h * a.group + row - node * a.group) * a.q_hs + piece * 8);
        }
        if (first)  // the copies wait for this: the first queries would otherwise queue behind all of the first keys and values
            asm volatile("bar.arrive 2, 384;" ::: "memory");
#pragma unroll
        for (int c = 0; c < LOADS; c++) {
            const int r = r0 + c * TOGETHER;
            uint4 v = q[c];
            v.x = (v.x ^ g.flip) & g.mask, v.y = (v.y ^ g.flip) & g.mask, v.z = (v.z ^ g.flip) & g.mask, v.w = (v.w ^ g.flip) & g.mask;
            *reinterpret_cast<uint4 *>(q_ptr + (r >> 7) * (128 * D * 2) + (r & 127) * 128 + (piece >> 3) * (128 * 128) + (((piece & 7) ^ (r & 7)) << 4)) = v;
        }
        fence_proxy_async();
        mbar_arrive(smem_addr(&x.q_ready));
    };
    TreeWalk<Shape::kUnitCost> ahead;
    ahead.begin(x);
    bool more = ahead.next(a, units);
    if (more)
        load_unit(ahead, true);
    while (more) {
        const TreeWalk<Shape::kUnitCost> walk = ahead;
        const int b = walk.b, h = walk.u / g.mtiles, n = walk.j1 - walk.j0, row = row_of(walk);
        const bool row_ok = row < a.rows;
        const int node = row_ok ? row / a.group : 0, head = h * a.group + (row_ok ? row % a.group : 0);
        const bool live = row_ok && node < walk.used;
        const bool warp_live = __any_sync(kFullMask, live);
        wait(x.q_ready, walk.seg);
        uint32_t anc[kTreeWords] = {};
        if (static_cast<int64_t>(walk.j1) * kTile > walk.context && live) {
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
        constexpr int HALVES = ROWT == 2 ? 2 : 1;  // of a tile that this group turns into weights
        for (int t = 0; t < n; t++, seen++) {
            const int odd = ROWT == 2 ? 0 : seen & 1;
            const uint32_t t_s = s_base + odd * kHalf;
            wait(x.s_ready[w][odd], ROWT == 2 ? seen : seen >> 1);
            uint64_t *p_ready = ROWT == 2 ? x.p_ready[w] : &x.p_ready[w][odd];
            if (!(warp_live && ok)) {
                __syncwarp();
                if ((tid & 31) == 0)
                    for (int half = 0; half < HALVES; half++)
                        mbar_arrive(smem_addr(&p_ready[half]));
                continue;
            }
            tc_fence_after();
            uint32_t s[2][32];  // the scores of one half at a time
            tmem_load32(t_s, s[0]);
            tmem_load32(t_s + 32, s[1]);
            const int first_word = ROWT == 2 ? 0 : 2 * w;
            const int64_t t0 = static_cast<int64_t>(walk.j0 + t) * kTile + 32 * first_word;
            const uint32_t *there = &x.valid[(tile + t) & (kSlots - 1)][first_word];
            uint32_t all = there[0] & there[1];
            if (ROWT == 2)
                all &= there[2] & there[3];
            const bool masked = t0 + kHalf * HALVES > walk.context || all != 0xFFFFFFFFu;
            // scores of positions c * 32 .. of the group's share that the row does not attend become -inf
            auto mask = [&](uint32_t (&v)[32], int c) {
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
                see = live ? see & there[c] : 0u;
#pragma unroll
                for (int e = 0; e < 32; e++)
                    v[e] = see >> e & 1u ? v[e] : 0xFF800000u;
            };
            float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            auto highest = [&](const uint32_t (&v)[32]) {
#pragma unroll
                for (int e = 0; e < 32; e++)
                    top[e & 3] = fmaxf(top[e & 3], __uint_as_float(v[e]));
            };
            tmem_wait_load();
            tmem_settle32(s[0]);
            tmem_settle32(s[1]);
            if (masked) {
                mask(s[0], 0);
                mask(s[1], 1);
            }
            highest(s[0]);
            highest(s[1]);
            if (ROWT == 2) {  // the maximum of the second half too: one reference a tile, while no product is under way
#pragma unroll 1
                for (int c = 2; c < 4; c++) {
                    uint32_t v[32];
                    tmem_load32(t_s + 32 * c, v);
                    tmem_wait_load();
                    tmem_settle32(v);
                    if (masked)
                        mask(v, c);
                    highest(v);
                }
            }
            const float m_tile = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * g.scale;
            if (__any_sync(kFullMask, m_tile > m_ref + kGrow)) {
                // (also the first tile of a unit: m_ref = -inf, nothing to rescale yet)
                const float m_new = fmaxf(m_ref, m_tile), keep = m_ref == m_new ? 1.0f : exp2_approx(m_ref - m_new);
                m_ref = m_new;
                l *= keep;
                if (t > 0) {
                    if (ROWT == 1)
                        wait_weighed(seen - 1);  // with one S a group it lies before this S in any case
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < D / 32; c++) {
                        uint32_t o[32];
                        tmem_load32(t_o + 32 * c, o);
                        tmem_wait_load();
                        tmem_settle32(o);
#pragma unroll
                        for (int e = 0; e < 32; e++)
                            o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                        tmem_store32(t_o + 32 * c, o);
                    }
                }
            }
            const float off = (m_ref == -INFINITY ? 0.0f : m_ref) - kBias;
#pragma unroll 1
            for (int half = 0; half < HALVES; half++) {
                if (half > 0) {
                    tmem_load32(t_s + kHalf, s[0]);
                    tmem_load32(t_s + kHalf + 32, s[1]);
                    tmem_wait_load();
                    tmem_settle32(s[0]);
                    tmem_settle32(s[1]);
                    if (masked) {
                        mask(s[0], 2);
                        mask(s[1], 3);
                    }
                }
                float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                uint32_t p[32];
#pragma unroll
                for (int e = 0; e < 32; e++) {
                    const int c = e >> 4, at = (e & 15) * 2;
                    const float p0 = exp2_approx(fmaf(__uint_as_float(s[c][at]), g.scale, -off));
                    const float p1 = exp2_approx(fmaf(__uint_as_float(s[c][at + 1]), g.scale, -off));
                    sum[(e & 1) * 2] += p0;
                    sum[(e & 1) * 2 + 1] += p1;
                    p[e] = TcType<T>::pack(p0, p1);
                }
                tmem_store32(t_s + half * kHalf, p);
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                tmem_wait_store();
                tc_fence_before();
                __syncwarp();
                if ((tid & 31) == 0)
                    mbar_arrive(smem_addr(&p_ready[half]));
            }
        }

        // ---- the unit's rows, or this CTA's part of them ----
        // a padding node's row took part with zeros where the tile was not masked: it attends nothing
        l = live ? l : 0.0f;
        float m = m_ref == -INFINITY || !live ? -INFINITY : m_ref - kBias;
        if (ROWT == 1)
            x.ml[w][trow] = make_float2(m, l);
        // every S of the unit has been read: the next unit's queries may take the place of its queries
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (tid == 0 && walk.seg > 0)
            x.bad[(walk.seg - 1) & (kSlots - 1)] = 0;  // the epilogue before is over
        float f0 = 1.0f, f1 = 0.0f;
        constexpr int COLS = ROWT == 2 ? D : D / 2;  // a group's columns of the output
        if (ROWT == 1) {
            const float2 u0 = x.ml[0][trow], u1 = x.ml[1][trow];
            m = fmaxf(u0.x, u1.x);
            const float base = m == -INFINITY ? 0.0f : m;
            f0 = exp2_approx(u0.x - base);
            f1 = exp2_approx(u1.x - base);
            l = u0.y * f0 + u1.y * f1;
        }
        more = ahead.next(a, units);
        if (more)
            load_unit(ahead, false);
        if (ROWT == 1 && seen > 1)
            wait_weighed(seen - 2);
        wait_weighed(seen - 1);
        if (ROWT == 1) {  // each group reads the other's sums too
            tc_fence_before();
            asm volatile("bar.sync 1, 256;" ::: "memory");
        }
        tc_fence_after();
        const bool whole = walk.whole();
        const int64_t slot = static_cast<int64_t>(blockIdx.x) * 2 + !walk.first;
        const int part_row = (ROWT == 2 ? w * 128 : 0) + trow;
        T *o_row = static_cast<T *>(a.out) + b * a.o_bs + node * a.o_ns + head * a.o_hs;
        const bool empty = l == 0.0f;
        const float inv = empty ? 0.0f : 1.0f / l;
        const bool broken = *reinterpret_cast<volatile int *>(&x.bad[walk.seg & (kSlots - 1)]) != 0;
        if (__any_sync(kFullMask, row_ok)) {
#pragma unroll 1  // code that runs once a unit: its fetch is what it costs
            for (int c = 0; c < COLS / 32; c++) {
                const int col = (ROWT == 2 ? 0 : w * COLS) + 32 * c;
                uint32_t o[32];
                if (ROWT == 2) {
                    tmem_load32(t_o + col, o);
                    tmem_wait_load();
                    tmem_settle32(o);
                } else {
                    const uint32_t o0 = x.tmem + lanes + 4 * kHalf + col;
                    tmem_load32(o0, o);
                    tmem_wait_load();
                    tmem_settle32(o);
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        o[i] = __float_as_uint(__uint_as_float(o[i]) * f0);
                    uint32_t o2[32];
                    tmem_load32(o0 + D, o2);
                    tmem_wait_load();
                    tmem_settle32(o2);
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        o[i] = __float_as_uint(fmaf(__uint_as_float(o2[i]), f1, __uint_as_float(o[i])));
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
                        for (int i = 0; i < 32; i += 4)  // [column / 4][row][4]: the lanes' stores are neighbours
                            *reinterpret_cast<uint4 *>(a.part_o + ((slot * (D / 4) + (col + i) / 4) * (ROWT * 128) + part_row) * 4) =
                                make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    }
                }
                __syncwarp();
            }
            if (row_ok && (ROWT == 2 || w == 0)) {
                if (!whole)
                    a.part_ml[slot * (ROWT * 128) + part_row] = make_float2(m, l);
                else if (a.lse)
                    a.lse[(static_cast<int64_t>(b) * a.nodes + node) * a.q_heads + head] = empty ? -INFINITY : (m + log2f(l)) * kLn2;
            }
        }
        tile += n;
        tc_fence_before();  // the next unit's products may overwrite what was read
        if (ROWT == 1)
            asm volatile("bar.sync 1, 256;" ::: "memory");
    }
}

template <typename T, int D, int ROWT>
__global__ void __launch_bounds__(kMmaThreads, 1) tree_attention_mma_kernel(const TreeMmaArgs g, const __grid_constant__ CUtensorMap k_map,
                                                                       const __grid_constant__ CUtensorMap v_map) {
    using Shape = TreeMmaShape<D, ROWT>;
    extern __shared__ __align__(1024) unsigned char smem[];
    TreeMmaExtras &x = *reinterpret_cast<TreeMmaExtras *>(smem + Shape::kQ + Shape::kRing * Shape::kBuffer);
    const TreeArgs &a = g.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int units = a.kv_heads * g.mtiles;
    auto places = [&](int tiles) { return static_cast<int64_t>(tiles + Shape::kUnitCost) * units; };

    if (tid == 0) {
        for (int i = 0; i < 8; i++) {
            mbar_init(smem_addr(&x.full[i]), 4);   // a copy warp each
            mbar_init(smem_addr(&x.empty[i]), 1);
        }
        for (int i = 0; i < 2; i++) {
            for (int k = 0; k < 2; k++) {
                mbar_init(smem_addr(&x.s_ready[i][k]), 1);
                mbar_init(smem_addr(&x.p_ready[i][k]), 4);  // a softmax warp each
                mbar_init(smem_addr(&x.pv_done[i][k]), 1);
            }
        }
        mbar_init(smem_addr(&x.q_ready), 256);
        mbar_init(smem_addr(&x.done), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        x.abort = 0;
        x.left = 0;
        for (int i = 0; i < kSlots; i++)
            x.bad[i] = 0;
    }
    int64_t lo, hi;
    if (g.whole) {  // this CTA's range of the units
        const int64_t total = static_cast<int64_t>(a.batch) * units;
        lo = blockIdx.x * total / kMmaCtas, hi = (blockIdx.x + 1) * total / kMmaCtas;
        if (tid == 0) {
            x.begin_b = static_cast<int>(lo / units);
            x.begin_u = static_cast<int>(lo % units);
            x.begin_j = 0;
            x.left = 1ll << 60;
            x.units_left = static_cast<int>(hi - lo);
        }
    } else {  // this CTA's range of the list of all tiles
        int64_t *s_scan = reinterpret_cast<int64_t *>(smem);
        const int per = (a.batch + kMmaThreads - 1) / kMmaThreads;
        const int b0 = min(a.batch, tid * per), b1 = min(a.batch, b0 + per);
        int64_t sum = 0;
        int tiles0 = 0;  // of this thread's first sequence
        for (int b = b0; b < b1; b++) {
            const int tiles = tree_tiles(a, b);
            tiles0 = b == b0 ? tiles : tiles0;
            sum += places(tiles);
        }
        int64_t upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(kFullMask, upto, o);
            upto += lane >= o ? v : 0;
        }
        if (lane == 31)
            s_scan[warp] = upto;
        __syncthreads();
        int64_t total = 0, before = upto - sum;
        for (int i = 0; i < kMmaThreads / 32; i++) {
            before += i < warp ? s_scan[i] : 0;
            total += s_scan[i];
        }
        lo = blockIdx.x * total / kMmaCtas, hi = (blockIdx.x + 1) * total / kMmaCtas;
        if (blockIdx.x == 0) {
            int64_t at = before;
            for (int b = b0; b < b1; b++) {
                g.starts[b] = at;
                at += places(b == b0 ? tiles0 : tree_tiles(a, b));
            }
            if (tid == 0)
                g.starts[a.batch] = total;
        }
        if (lo < hi && lo >= before && lo < before + sum) {
            int64_t at = before;
            int b = b0, tiles = tiles0;
            while (lo >= at + places(tiles)) {
                at += places(tiles);
                tiles = tree_tiles(a, ++b);
            }
            x.begin_b = b;
            const int one = tiles + Shape::kUnitCost;
            const int64_t into = lo - at;
            x.begin_u = into >> 32 ? static_cast<int>(into / one) : static_cast<int>(static_cast<uint32_t>(into) / static_cast<uint32_t>(one));
            x.begin_j = static_cast<int>(into - static_cast<int64_t>(x.begin_u) * one);
            x.left = hi - lo;
            x.units_left = 0x7FFFFFFF;
        }
    }
    if (lo >= hi)
        return;  // less work than CTAs
    if (warp == kProductWarp)
        tmem_alloc(smem_addr(&x.tmem), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t q_smem = smem_addr(smem), ring = q_smem + Shape::kQ;

    if (warp < 8)
        tree_softmax_role<T, D, ROWT>(g, x, smem, units);
    else if (warp < 12)
        tree_copy_role<T, D, ROWT>(g, &k_map, &v_map, x, ring, units);
    else if (warp == kProductWarp)
        tree_product_role<T, D, ROWT>(g, x, q_smem, ring, units);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kProductWarp)
        tmem_free(x.tmem, 512);
}

// ---- join: a unit that several CTAs worked on; a thread takes a row's D / 8 neighbouring columns, so that a warp reads the
// parts of 32 rows as they lie; parts are added in the order of the CTAs ----
constexpr int kMmaJoinRows = 32;

template <typename T, int D, int ROWT>
__global__ void __launch_bounds__(kMmaJoinRows * 8) tree_attention_mma_join_kernel(const TreeMmaArgs g) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr int COLS = D / 8;
    const TreeArgs &a = g.a;
    const int units = a.kv_heads * g.mtiles, b = blockIdx.x / units, u = blockIdx.x % units;
    const int in_unit = blockIdx.y * kMmaJoinRows + (threadIdx.x & 31), col = (threadIdx.x >> 5) * COLS;
    const int row = u % g.mtiles * (ROWT * 128) + in_unit;
    const int64_t total = g.starts[a.batch], begin = g.starts[b], places = (g.starts[b + 1] - begin) / units;
    const int64_t lo = begin + u * places, hi = lo + places - TreeMmaShape<D, ROWT>::kUnitCost;  // the unit's tiles
    const int c0 = static_cast<int>(((lo + 1) * kMmaCtas - 1) / total), c1 = static_cast<int>((hi * kMmaCtas - 1) / total);
    if (c0 == c1)
        return;  // written out by the one CTA
    float top = -INFINITY, l = 0.0f, acc[COLS];
#pragma unroll
    for (int e = 0; e < COLS; e++)
        acc[e] = 0.0f;
    __shared__ int s_slot[32];
    __shared__ float2 s_ml[32][kMmaJoinRows];
    const int lane = threadIdx.x & 31;
    for (int c = c0; c <= c1; c += 32) {  // 32 parts at a time
        const int count = min(32, c1 - c + 1);
        if (static_cast<int>(threadIdx.x) < count) {
            const int64_t at = c + threadIdx.x, from = at * total / kMmaCtas;
            // the CTA's first slot when its range begins inside the unit; an empty range has none
            s_slot[threadIdx.x] = from == (at + 1) * total / kMmaCtas ? -1 : static_cast<int>(at * 2 + (from < lo));
        }
        __syncthreads();
        for (int p = threadIdx.x >> 5; p < count; p += 8)
            s_ml[p][lane] = s_slot[p] >= 0 && row < a.rows ? a.part_ml[static_cast<int64_t>(s_slot[p]) * (ROWT * 128) + in_unit] : make_float2(-INFINITY, 0.0f);
        __syncthreads();
        float higher = top;
        for (int p = 0; p < count; p++)
            higher = fmaxf(higher, s_ml[p][lane].x);
        const float base = higher == -INFINITY ? 0.0f : higher, keep = exp2_approx(top - base);
        top = higher;
        l *= keep;
#pragma unroll
        for (int e = 0; e < COLS; e++)
            acc[e] *= keep;
#pragma unroll 2
        for (int p = 0; p < count; p++) {
            const int slot = s_slot[p];
            if (slot < 0 || row >= a.rows)
                continue;
            const float4 *o = reinterpret_cast<const float4 *>(a.part_o) + (static_cast<int64_t>(slot) * (D / 4) + col / 4) * (ROWT * 128) + in_unit;
            const float f = exp2_approx(s_ml[p][lane].x - base);
            l = fmaf(f, s_ml[p][lane].y, l);
#pragma unroll
            for (int e = 0; e < COLS / 4; e++) {
                const float4 v = o[e * (ROWT * 128)];
                acc[4 * e] = fmaf(f, v.x, acc[4 * e]);
                acc[4 * e + 1] = fmaf(f, v.y, acc[4 * e + 1]);
                acc[4 * e + 2] = fmaf(f, v.z, acc[4 * e + 2]);
                acc[4 * e + 3] = fmaf(f, v.w, acc[4 * e + 3]);
            }
        }
        __syncthreads();
    }
    if (row >= a.rows)
        return;
    const int node = row / a.group, head = u / g.mtiles * a.group + row % a.group;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T *out = static_cast<T *>(a.out) + b * a.o_bs + node * a.o_ns + head * a.o_hs + col;
#pragma unroll
    for (int e = 0; e < COLS; e += 8) {
        uint32_t v[4];
#pragma unroll
        for (int k = 0; k < 4; k++)
            v[k] = l == 0.0f ? 0u : TcType<T>::pack(acc[e + 2 * k] * inv, acc[e + 2 * k + 1] * inv);
        *reinterpret_cast<uint4 *>(out + e) = make_uint4(v[0], v[1], v[2], v[3]);
    }
    if (a.lse && col == 0)
        a.lse[(static_cast<int64_t>(b) * a.nodes + node) * a.q_heads + head] = l == 0.0f ? -INFINITY : (top + log2f(l)) * kLn2;
}

// ---- host side ----
bool tree_mma_serves(const vkop_tree_attention_desc &d) {
    return d.dtype != VKOP_F32 && (d.head_dim == 64 || d.head_dim == 128);
}

static int64_t slot_rows(const TreeArgs &a) { return a.rows > 128 ? 256 : 128; }

// Whole units or an even share of all tiles?  The scan, the parts and the join cost about as much as 11 tiles, a change of
// units as 3; whole units leave some CTAs with one more than others.  Measured, us in a graph, whole against shared (8 cache
// heads of 128, bf16): 1 sequence of 1 / 4 / 8 tiles 9.1 / 12.5 / 17.0 against 11.9 / 15.8 / 17.6, 16 sequences of 8 tiles
// 18.6 against 28.5, 64 sequences of 8 tiles 76 against 85.  Lengths beyond 16 tiles may differ too much within a batch.
static bool whole_units(const vkop_tree_attention_desc &d) {
    const int64_t longest = (d.max_context > 0 ? d.max_context : static_cast<int64_t>(d.max_pages) * d.page_size) + d.nodes;
    const int64_t tiles = (longest + kTile - 1) / kTile, rows = static_cast<int64_t>(d.nodes) * (d.q_heads / d.kv_heads);
    const int64_t units = d.batch * d.kv_heads * (rows > 128 ? (rows + 255) / 256 : 1);
    return tiles <= 16 && (units + kMmaCtas - 1) / kMmaCtas * (tiles + 3) * kMmaCtas <= units * (tiles + 3) + 11 * kMmaCtas;
}

size_t tree_mma_workspace(const vkop_tree_attention_desc &d) {
    if (whole_units(d))
        return 0;
    const int64_t rows = static_cast<int64_t>(d.nodes) * (d.q_heads / d.kv_heads) > 128 ? 256 : 128;
    const size_t starts = (static_cast<size_t>(d.batch + 1) * 8 + 31) / 32 * 32 + 32;
    return starts + static_cast<size_t>(kMmaCtas) * 2 * rows * (d.head_dim + 2) * sizeof(float);
}

template <typename T, int D, int ROWT>
static int launch_mma_t(const TreeMmaArgs &g, const CUtensorMap *maps, cudaStream_t stream) {
    constexpr int smem = TreeMmaShape<D, ROWT>::kSmem;
    static std::atomic<uint64_t> ready{0};  // devices whose kernel has been given its shared memory
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess)
        return VKOP_CUDA_ERROR;
    const uint64_t bit = device < 64 ? 1ull << device : 0;
    if (!(ready.load(std::memory_order_relaxed) & bit)) {
        if (cudaFuncSetAttribute(tree_attention_mma_kernel<T, D, ROWT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
            cudaGetLastError();
            return VKOP_CUDA_ERROR;
        }
        ready.fetch_or(bit, std::memory_order_relaxed);
    }
    tree_attention_mma_kernel<T, D, ROWT><<<kMmaCtas, kMmaThreads, smem, stream>>>(g, maps[0], maps[1]);
    note_launch();
    if (check_launch() != VKOP_OK)
        return VKOP_CUDA_ERROR;
    if (g.whole)
        return VKOP_OK;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(g.a.batch * g.a.kv_heads * g.mtiles),
                       static_cast<unsigned>((min(g.a.rows, ROWT * 128) + kMmaJoinRows - 1) / kMmaJoinRows));
    cfg.blockDim = dim3(kMmaJoinRows * 8);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, tree_attention_mma_join_kernel<T, D, ROWT>, g) != cudaSuccess) {
        cudaGetLastError();
        return VKOP_CUDA_ERROR;
    }
    note_launch();
    return VKOP_OK;
}

template <typename T>
static int launch_mma_type(const TreeMmaArgs &g, const CUtensorMap *maps, cudaStream_t stream) {
    if (g.a.head_dim == 64)
        return g.a.rows > 128 ? launch_mma_t<T, 64, 2>(g, maps, stream) : launch_mma_t<T, 64, 1>(g, maps, stream);
    return g.a.rows > 128 ? launch_mma_t<T, 128, 2>(g, maps, stream) : launch_mma_t<T, 128, 1>(g, maps, stream);
}

// The cache as a tensor [page, head, slot, element] for copies of `rows` x 64 elements.  False where the driver has no such map.
static bool cache_map(CUtensorMap *map, int dtype, const void *base, int64_t num_pages, int64_t ps, int64_t ts, int64_t hs, const TreeArgs &a, int rows) {
    using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            fn = nullptr;
        }
        return reinterpret_cast<Encode>(fn);
    }();
    if (!encode)
        return false;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(a.head_dim), static_cast<cuuint64_t>(a.page_size), static_cast<cuuint64_t>(a.kv_heads),
                                static_cast<cuuint64_t>(num_pages)};
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(ts) * 2, static_cast<cuuint64_t>(hs) * 2, static_cast<cuuint64_t>(ps) * 2};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(rows), 1, 1}, steps[4] = {1, 1, 1, 1};
    return encode(map, dtype == VKOP_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(base), dims, strides,
                  box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int launch_tree_mma(const TreeArgs &args, const vkop_tree_attention_desc &d, void *workspace, cudaStream_t stream) {
    const int dtype = d.dtype;
    TreeMmaArgs g;
    g.a = args;
    g.whole = whole_units(d);
    workspace = reinterpret_cast<void *>((reinterpret_cast<uintptr_t>(workspace) + 31) / 32 * 32);
    g.starts = static_cast<int64_t *>(workspace);
    const size_t starts = (static_cast<size_t>(args.batch + 1) * 8 + 31) / 32 * 32;
    g.a.part_ml = reinterpret_cast<float2 *>(static_cast<char *>(workspace) + starts);
    g.a.part_o = reinterpret_cast<float *>(g.a.part_ml + kMmaCtas * 2 * slot_rows(args));
    g.mtiles = args.rows > 128 ? (args.rows + 255) / 256 : 1;
    g.scale = args.scale_log2 == 0.0f ? 1.0f : fabsf(args.scale_log2);
    g.mask = args.scale_log2 == 0.0f ? 0u : 0xFFFFFFFFu;
    g.flip = args.scale_log2 < 0.0f ? 0x80008000u : 0u;
    g.page_shift = (args.page_size & (args.page_size - 1)) == 0 ? __builtin_ctz(static_cast<unsigned>(args.page_size)) : -1;
    CUtensorMap maps[2] = {};
    g.box_rows = 0;
    // boxes of the largest power of two that divides the page size: tiles begin at multiples of it, so none crosses a page
    const int divides = args.page_size & -args.page_size, rows = divides < 32 ? divides : 32;
    if (rows >= 8 && args.max_pages > 0) {
        if (cache_map(&maps[0], dtype, args.k, args.num_pages, args.k_ps, args.k_ts, args.k_hs, args, rows) &&
            cache_map(&maps[1], dtype, args.v, args.num_pages, args.v_ps, args.v_ts, args.v_hs, args, rows))
            g.box_rows = rows;
    }
    return dtype == VKOP_F16 ? launch_mma_type<__half>(g, maps, stream) : launch_mma_type<__nv_bfloat16>(g, maps, stream);
}

}  // namespace vkop_cuda
