// Products with 4-bit weights (w4.cuh has the format) on the tcgen05 tensor path, for more rows than the few of w4.cu:
// out[M, N] = (act(x W^T + bias) + residual) * out_scale.
//
// The WEIGHT rows are the 128 rows of the MMA and the rows of x its columns (BT of them, any multiple of 16 up to 256), so a
// few dozen rows of x waste nothing. The weights never exist in memory as fp16: warps unpack them in registers and write
// them to TENSOR MEMORY, from where the MMA reads its A operand; shared memory carries the 4-bit codes and x only. One
// persistent CTA per SM, twenty warps:
//   * warps 0-11 unpack, in three groups that take turns over units of 128 k: a warp owns 32 weight rows (its TMEM lane
//     quarter, one row per thread), 64 bytes of codes from shared memory, 64 fp16 pairs to TMEM (tcgen05.st);
//   * warps 12-15: epilogue, one weight row per thread; for each row of x a warp stores 32 consecutive outputs (64 bytes). At
//     a CTA's last tile the unpacking warps help;
//   * warp 16: TMA loads of x (128-byte swizzle); warp 18: TMA loads of codes (64-byte swizzle); rings of their own, so that
//     either stream runs ahead of the A stages (with x in the stages of A, of which there are three beside two accumulators
//     of 160 columns, its latency set the pace);
//   * warp 19: scales and zero points of 1024 k at a time, gathered into shared memory as fp16 (64 * scale);
//   * warp 17: tcgen05.mma, D[128 x BT] += A[TMEM] B[x].
// K split (SPLIT), where there are fewer tiles than SMs: a cluster of 2, 4 or 8 CTAs shares a tile, each multiplies a part of K,
// and for every 16 rows of x one of them receives the others' sums in its shared memory and adds them in rank order.
// CTA pairs (PAIR): the MMA covers 256 weight rows, 128 from each CTA's tensor memory, and each CTA loads half of x's tile:
// per 64 k an SM then fetches BT * 64 + 4096 bytes instead of BT * 128 + 4096, where L2 was the bound.
//
// Measured (rows x N x K): 154 x 166400 x 2048 88 us = 1190 TFLOP/s (1374 is cuBLAS's sustained rate),
// the tensor pipe 69% busy; 2048 x 1280 x 5120 with a residual 24.4 us, 77 x 5120 x 1280 8.4 us, of which 5 us are what any
// launch of this kernel takes (set-up, first loads, the fill of the rings and the epilogue: 77 x 1280 x 256 takes 5.0 us).
// Bound, where there are tiles for all SMs, by tensor pipe and unpacking together, which take about equally long.
//
// Every mbarrier wait is bounded (tc05.cuh): on a time-out the CTA records a status word, stops storing, frees its TMEM and
// returns; the host reads the word with katz_tc05_status().
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "tc05.cuh"
#include "w4.cuh"
#include "katz_b200.h"

namespace katz {

using namespace tc05;
using namespace w4;

int* tc05_status_device_ptr();   // defined next to the status word (gemm_tc05.cu)

constexpr int WT_THREADS = 640;
constexpr int WT_GROUPS = 3, WT_GROUP_WARPS = 4;               // unpacking warps
constexpr int WT_UNPACK_WARPS = WT_GROUPS * WT_GROUP_WARPS;
constexpr int WT_EPILOGUE = WT_UNPACK_WARPS, WT_X = WT_EPILOGUE + 4, WT_MMA = WT_X + 1, WT_Q = WT_X + 2, WT_S = WT_X + 3;   // first warp of each role
constexpr int WT_XS = 8, WT_AS = 6, WT_QS = 6, WT_SS = 2;      // stages of each ring (x and A: at most)
// A barrier's parity tells a group that the use before its own is over only if the group knows that the one before THAT is:
// of A's stages it knows that unit n - WT_GROUPS - stages has been multiplied (its last wait), and must know it of n - 2
// stages; of the codes' stages it knows the loads of its own units only, n - WT_GROUPS i, and must know that of n - WT_QS.
static_assert(WT_QS % WT_GROUPS == 0, "the unit that used a stage of codes before must be one of the same group");
constexpr int WT_Q_BYTES = 128 * 64;                           // 128 rows x 128 k of codes
constexpr int WT_S_UNITS = 8, WT_S_ROWS = WT_S_UNITS * 128 / 32;      // a scale block: units of 128 k, groups at most
constexpr int WT_SCALE_BYTES = WT_S_ROWS * 128 * 2, WT_ZERO_BYTES = WT_S_ROWS * 128;
constexpr int WT_TMEM_COLS = 512;
constexpr int WT_BARS = 2 * (WT_XS + WT_QS + WT_AS + WT_SS + 2) + 2;
constexpr int WT_FIXED_SMEM = WT_QS * WT_Q_BYTES + WT_SS * (WT_SCALE_BYTES + WT_ZERO_BYTES) + WT_BARS * 8 + 16 + 1024;
constexpr int WT_MAX_SMEM = 232448;

struct W4Tile {
    int bt, acc_stride, n_acc;                 // columns of a tile (rows of x), of an accumulator buffer; buffers
    int x_stages, x_bytes, a_stages;           // x_bytes: of x in a stage of this CTA (two boxes of 64 k)
    int m_tiles, n_tiles;                      // n_tiles: of 128 rows, of a pair's 256
    int split;                                 // CTAs that share a tile (SPLIT)
    bool in_pairs;                             // out (and residual) allow 4-byte accesses to (n, n + 1), n even
    int* status;
};

// One word (8 codes, k = 0..7) -> 64 * weight as four fp16 pairs in k order. Byte i of the word is copied into both halves;
// the low half keeps its low four bits (1024 + code), the high half its high four (1024 + 16 code, times 1/16).
__device__ __forceinline__ void weights8_in_order(uint32_t w, __half2 minus, __half2 scale, uint32_t* o) {
    const __half2 mul = as_half2(0x2c003c00u);      // (1, 1/16)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t both = __byte_perm(w, 0, 0x4040 + 0x0101 * i);
        const __half2 d = __hfma2(as_half2(and_or_1024<0x00f0000fu>(both)), mul, minus);
        o[i] = as_u32(__hmul2(d, scale));
    }
}

// Shared memory by 32-bit address: the aligned base of dynamic shared memory is an integer to the compiler, and through a
// pointer made of it every access would be a generic one with 64-bit arithmetic.
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
    unsigned short v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ float lds_f32(uint32_t a) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void sts16(uint32_t a, __half v) { asm volatile("st.shared.u16 [%0], %1;" ::"r"(a), "h"(__half_as_ushort(v)) : "memory"); }
__device__ __forceinline__ void sts8(uint32_t a, uint32_t v) { asm volatile("st.shared.u8 [%0], %1;" ::"r"(a), "r"(v) : "memory"); }

// position in a ring of `n` stages
struct Ring {
    uint32_t s = 0, phase = 0;
    __device__ __forceinline__ void next(uint32_t n) {
        if (++s == n) {
            s = 0;
            phase ^= 1;
        }
    }
    __device__ __forceinline__ void skip(uint32_t k, uint32_t n) {      // k <= n
        s += k;
        if (s >= n) {
            s -= n;
            phase ^= 1;
        }
    }
};

template <bool PAIR, bool SPLIT>
__global__ void __launch_bounds__(WT_THREADS, 1) linear_w4_tc05_kernel(const __grid_constant__ CUtensorMap tmX,
                                                                       const __grid_constant__ CUtensorMap tmQ, const W4Params p,
                                                                       const W4Tile t) {
    extern __shared__ unsigned char smem_raw[];
    const uint32_t smem = (smem_u32(smem_raw) + 1023) & ~1023u;
    const uint32_t q_ring = smem + t.x_stages * t.x_bytes, s_ring = q_ring + WT_QS * WT_Q_BYTES, z_ring = s_ring + WT_SS * WT_SCALE_BYTES,
                   bars = z_ring + WT_SS * WT_ZERO_BYTES, tmem_slot = bars + WT_BARS * 8,
                   sums = tmem_slot + 16;      // SPLIT: [16-row chunk of mine][other rank][16][128] floats
    const uint32_t q_full = bars, q_empty = q_full + 8 * WT_QS,
                   a_full = q_empty + 8 * WT_QS, a_empty = a_full + 8 * WT_AS, s_full = a_empty + 8 * WT_AS,
                   s_empty = s_full + 8 * WT_SS, acc_full = s_empty + 8 * WT_SS, acc_empty = acc_full + 16, x_full = acc_empty + 16, x_empty = x_full + 8 * WT_XS,
                   last_full = x_empty + 8 * WT_XS;      // the last tile has a barrier of its own: warps that skipped acc_full cannot tell its parity
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    static_assert(!(PAIR && SPLIT), "a cluster is a pair or a split of K");
    const uint32_t rank = PAIR ? cluster_ctarank() : 0, part = SPLIT ? cluster_ctarank() : 0;
    constexpr int CTAS = PAIR ? 2 : 1;

    if (threadIdx.x == 0) {
        for (int i = 0; i < WT_XS; ++i) {
            mbar_init(x_full + 8 * i, 1);
            mbar_init(x_empty + 8 * i, 1);
        }
        for (int i = 0; i < WT_QS; ++i) {
            mbar_init(q_full + 8 * i, 1);
            mbar_init(q_empty + 8 * i, WT_GROUP_WARPS);
        }
        for (int i = 0; i < WT_AS; ++i) {
            mbar_init(a_full + 8 * i, WT_GROUP_WARPS * CTAS);
            mbar_init(a_empty + 8 * i, 1);
        }
        for (int i = 0; i < WT_SS; ++i) {
            mbar_init(s_full + 8 * i, 1);
            mbar_init(s_empty + 8 * i, WT_UNPACK_WARPS);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(acc_full + 8 * i, 1);
            mbar_init(acc_empty + 8 * i, 4 * CTAS);
        }
        mbar_init(last_full, 1);
        fence_barrier_init();
        tma_prefetch_desc(&tmX);
        tma_prefetch_desc(&tmQ);
    }
    if (warp == WT_MMA) {
        if (PAIR) {
            tmem_alloc_pair(tmem_slot, WT_TMEM_COLS);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(tmem_slot, WT_TMEM_COLS);
            tmem_relinquish();
        }
    }
    fence_before_sync();
    __syncthreads();
    if (PAIR) cluster_sync_all();      // the peer's barriers are initialised before anything signals them
    if (SPLIT) cluster_arrive_relaxed();      // this CTA runs; waited for before the first write to another's shared memory
    fence_after_sync();
    uint32_t tmem_base;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot) : "memory");
    const uint32_t a_base = tmem_base + t.n_acc * t.acc_stride;

    const int all_units = (p.K + 127) >> 7;      // stages of 128 k; this CTA's: units from first_unit on
    const int first_unit = SPLIT ? (int)part * all_units / t.split : 0;
    const int units = SPLIT ? ((int)part + 1) * all_units / t.split - first_unit : all_units;
    const int total = t.m_tiles * t.n_tiles;
    const int per_item = SPLIT ? t.split : CTAS;
    const int item0 = (int)blockIdx.x / per_item, item_stride = (int)gridDim.x / per_item;
    auto rows_of = [&](int tile, int& m0, int& n0) {      // weight rows fastest: CTAs at work at one time share x
        const int mt = tile / t.n_tiles;
        m0 = mt * t.bt;
        n0 = (tile - mt * t.n_tiles) * 128 * CTAS + 128 * (int)rank;
    };
    const int last = item0 < total ? item0 + (total - 1 - item0) / item_stride * item_stride : -1;      // this CTA's last tile
    // Nothing above touches global memory; every role waits for the kernels this launch depends on before it goes on (those
    // that read none as well: their bounded waits must not run out while a predecessor still runs).
    pdl_wait();
    pdl_launch_dependents();

    bool ok = true;
    if (warp < WT_UNPACK_WARPS) {
        // ---------------------------------------------------------------------------------------- unpack
        const int quarter = warp & 3, group = warp >> 2;
        const int row = quarter * 32 + lane;
        const uint32_t a_mine = a_base + ((uint32_t)(quarter * 32) << 16);
        const uint32_t swz = (uint32_t)((row >> 1) & 3) << 4, q_mine = q_ring + row * 64;
        // The groups take turns over the CTA's units. A warp has its next unit's codes in registers before it hands over the
        // current one, and polls the two barriers it will need once before the arithmetic, so that a barrier that has long
        // been passed (the usual case) costs nothing. (Waiting where the data was needed, a warp took 1800 cycles for 330
        // of arithmetic.)
        // A stage of codes goes back to TMA when its unit is in tensor memory, not when its loads have been issued: an arrival does
        // not wait for shared-memory loads in flight, and where they were delayed TMA's next write overtook them (147 x 3663 x
        // 7168: in one call of thirty a weight row had the codes of six units later).
        Ring q, a, sc;
        q.skip(group, WT_QS);
        a.skip(group, t.a_stages);
        const int count = item0 < total ? ((total - 1 - item0) / item_stride + 1) * units : 0;
        int now = 0, mine = group;      // this CTA's units so far; this warp's next one
        uint4 v0, v1, v2, v3;
        auto wait_all = [&](uint32_t bar, uint32_t phase) { return __all_sync(0xffffffffu, mbar_wait(bar, phase)); };
        auto codes = [&](uint32_t c) { return lds128(q_mine + q.s * WT_Q_BYTES + ((c << 4) ^ swz)); };
        if (mine < count) {
            ok = wait_all(q_full + 8 * q.s, q.phase);
            if (ok) v0 = codes(0), v1 = codes(1), v2 = codes(2), v3 = codes(3);
        }
        for (int tile = item0; tile < total && ok; tile += item_stride) {
            for (int u0 = 0; u0 < units && ok; u0 += WT_S_UNITS) {
                // every group waits for every scale block, so that none can be a whole ring ahead of another
                ok = wait_all(s_full + 8 * sc.s, sc.phase);
                const int u1 = min(u0 + WT_S_UNITS, units);
                const int first = u0 + (mine - now);
                for (int u = first; u < u1 && ok; u += WT_GROUPS) {
                    const bool more = mine + WT_GROUPS < count;
                    const uint32_t q_bar = 8 * q.s, a_bar = 8 * a.s, a_phase = a.phase ^ 1, ta = a_mine + 64 * a.s;
                    mine += WT_GROUPS;
                    q.skip(WT_GROUPS, WT_QS);
                    a.skip(WT_GROUPS, t.a_stages);
                    const bool a_free = mbar_test(a_empty + a_bar, a_phase);
                    const bool q_there = more && mbar_test(q_full + 8 * q.s, q.phase);
                    const uint32_t scales = s_ring + sc.s * WT_SCALE_BYTES + row * 2, zeros = z_ring + sc.s * WT_ZERO_BYTES + row;
                    const uint32_t k = (u - u0) * 128;
                    uint32_t w[32];
                    auto unpack = [&](uint32_t k32, const uint4& v, uint32_t* o) {      // 32 k of one group
                        const uint32_t j = ((k + 32 * k32) >> p.group_shift) * 128;
                        const __half2 scale = as_half2(lds16(scales + 2 * j) * 0x10001u);
                        uint32_t minus = 0xd480e408u;      // (-(1024 + 8), -(64 + 8))
                        if (p.zero) minus = 0xd400e400u + 0x00100001u * lds8(zeros + j);
                        weights8_in_order(v.x, as_half2(minus), scale, o);
                        weights8_in_order(v.y, as_half2(minus), scale, o + 4);
                        weights8_in_order(v.z, as_half2(minus), scale, o + 8);
                        weights8_in_order(v.w, as_half2(minus), scale, o + 12);
                    };
                    unpack(0, v0, w);
                    unpack(1, v1, w + 16);
                    if (!__all_sync(0xffffffffu, a_free)) {
                        ok = wait_all(a_empty + a_bar, a_phase);
                        if (!ok) break;
                    }
                    fence_after_sync();
                    tmem_st_32x32(ta, w);
                    const bool read_now = __all_sync(0xffffffffu, q_there);
                    if (read_now) v0 = codes(0), v1 = codes(1);
                    unpack(2, v2, w);
                    unpack(3, v3, w + 16);
                    tmem_st_32x32(ta + 32, w);
                    if (read_now) v2 = codes(2), v3 = codes(3);
                    tmem_st_wait();
                    fence_before_sync();
                    __syncwarp();
                    if (lane == 0) {
                        if (PAIR) mbar_arrive_cluster_tmem(mapa_shared(a_full + a_bar, 0));      // the leader's MMA thread waits for both CTAs
                        else mbar_arrive(a_full + a_bar);
                        mbar_arrive(q_empty + q_bar);
                    }
                    if (more && !read_now) {
                        ok = wait_all(q_full + 8 * q.s, q.phase);
                        if (!ok) break;
                        v0 = codes(0), v1 = codes(1), v2 = codes(2), v3 = codes(3);
                    }
                }
                now += u1 - u0;
                __syncwarp();
                if (lane == 0) mbar_arrive(s_empty + 8 * sc.s);
                sc.next(WT_SS);
            }
        }
        if (!ok && lane == 0) atomicCAS(t.status, 0, 21);
    } else if (warp == WT_X) {
        // ---------------------------------------------------------------------------------------- x
        if (elect_one()) {
            Ring x;
            uint32_t issued = 0;
            bool ok = true;
            for (int tile = item0; tile < total && ok; tile += item_stride) {
                int m0, n0;
                rows_of(tile, m0, n0);
                for (int u = 0; u < units; ++u) {
                    if (!mbar_wait_idle(x_empty + 8 * x.s, x.phase ^ 1)) { ok = false; break; }
                    const uint32_t dst = smem + x.s * t.x_bytes, half = t.x_bytes / 2;
                    const int k = (first_unit + u) * 128;
                    const bool two = k + 64 < p.K;      // a tile's last unit may be one box
                    if (PAIR) {
                        // both CTAs' bytes are counted on the leader's barrier, which the leader arms for both
                        const uint32_t bar = mapa_shared(x_full + 8 * x.s, 0);
                        const int m = m0 + (int)rank * (t.bt / 2);
                        if (rank == 0) mbar_expect_tx(x_full + 8 * x.s, two ? 2 * t.x_bytes : t.x_bytes);
                        tma_load_2d_pair(dst, &tmX, k, m, bar);
                        if (two) tma_load_2d_pair(dst + half, &tmX, k + 64, m, bar);
                    } else {
                        const uint32_t bar = x_full + 8 * x.s;
                        mbar_expect_tx(bar, two ? t.x_bytes : half);
                        tma_load_2d(dst, &tmX, k, m0, bar);
                        if (two) tma_load_2d(dst + half, &tmX, k + 64, m0, bar);
                    }
                    ++issued;
                    x.next(t.x_stages);
                }
            }
            if (!ok) {
                atomicCAS(t.status, 0, 23);
                // copies in flight land before the CTA's shared memory is released (a pair's second CTA waits for the first
                // in the cluster barrier of the teardown: its copies are counted on the leader's barriers)
                if (rank == 0) {
                    const uint32_t n = t.x_stages, first = issued > n ? issued - n : 0;
                    for (uint32_t i = first; i < issued; ++i) mbar_wait_idle(x_full + 8 * (i % n), (i / n) & 1);
                }
            }
        }
    } else if (warp == WT_MMA) {
        // ---------------------------------------------------------------------------------------- MMA
        if (rank == 0 && elect_one()) {
            const uint32_t idesc = idesc_f16(PAIR ? 256 : 128, t.bt);
            Ring x, a, acc;
            bool ok = true;
            for (int tile = item0; tile < total && ok; tile += item_stride) {
                if (!mbar_wait_idle(acc_empty + 8 * acc.s, acc.phase ^ 1)) { ok = false; break; }
                fence_after_sync();
                const uint32_t tacc = tmem_base + acc.s * t.acc_stride;
                for (int u = 0; u < units; ++u) {
                    // both barriers are looked at before either is waited for: one round trip where both have been passed
                    const bool a_there = mbar_test(a_full + 8 * a.s, a.phase), x_there = mbar_test(x_full + 8 * x.s, x.phase);
                    if (!(a_there && x_there) && !(mbar_wait_idle(a_full + 8 * a.s, a.phase) && mbar_wait_idle(x_full + 8 * x.s, x.phase))) { ok = false; break; }
                    fence_after_sync();
                    const uint32_t xs = smem + x.s * t.x_bytes, ta = a_base + 64 * a.s;
                    auto issue = [&](int b) {      // 64 k
                        const uint64_t bd = smem_desc_sw128(xs + b * (t.x_bytes / 2));
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            if (PAIR) umma_f16_ta_pair(tacc, ta + 32 * b + 8 * k, bd + 2 * k, idesc, (u | b | k) != 0);
                            else umma_f16_ta(tacc, ta + 32 * b + 8 * k, bd + 2 * k, idesc, (u | b | k) != 0);
                        }
                    };
                    issue(0);
                    if ((first_unit + u) * 128 + 64 < p.K) issue(1);
                    if (PAIR) {
                        umma_commit_pair(a_empty + 8 * a.s, 3);
                        umma_commit_pair(x_empty + 8 * x.s, 3);
                    } else {
                        umma_commit(a_empty + 8 * a.s);
                        umma_commit(x_empty + 8 * x.s);
                    }
                    a.next(t.a_stages);
                    x.next(t.x_stages);
                }
                if (ok) {
                    const uint32_t full = tile == last ? last_full : acc_full + 8 * acc.s;
                    if (PAIR) umma_commit_pair(full, 3);
                    else umma_commit(full);
                }
                acc.next(t.n_acc);
            }
            if (!ok) atomicCAS(t.status, 0, 24);
        }
    } else if (warp == WT_Q) {
        // ---------------------------------------------------------------------------------------- codes
        if (elect_one()) {
            Ring q;
            uint32_t issued = 0;
            bool ok = true;
            for (int tile = item0; tile < total && ok; tile += item_stride) {
                int m0, n0;
                rows_of(tile, m0, n0);
                for (int u = 0; u < units; ++u) {
                    if (!mbar_wait_idle(q_empty + 8 * q.s, q.phase ^ 1)) { ok = false; break; }
                    mbar_expect_tx(q_full + 8 * q.s, WT_Q_BYTES);
                    tma_load_2d(q_ring + q.s * WT_Q_BYTES, &tmQ, (first_unit + u) * 64, n0, q_full + 8 * q.s);
                    ++issued;
                    q.next(WT_QS);
                }
            }
            if (!ok) {
                atomicCAS(t.status, 0, 25);
                const uint32_t n = WT_QS, first = issued > n ? issued - n : 0;
                for (uint32_t i = first; i < issued; ++i) mbar_wait_idle(q_full + 8 * (i % n), (i / n) & 1);
            }
        }
    } else if (warp == WT_S) {
        // ---------------------------------------------------------------------------------------- scales, zero points
        Ring sc;
        bool ok = true;
        const int per_block = (WT_S_UNITS * 128) >> p.group_shift;
        const bool by_four = ((p.J | (first_unit * 128) >> p.group_shift) & 3) == 0 && ((uintptr_t)p.scale & 7) == 0;
        for (int tile = item0; tile < total && ok; tile += item_stride) {
            int m0, n0;
            rows_of(tile, m0, n0);
            const int j_end = min(p.J, ((first_unit + units) * 128) >> p.group_shift);
            for (int j0 = (first_unit * 128) >> p.group_shift; j0 < j_end; j0 += per_block) {
                ok = __all_sync(0xffffffffu, mbar_wait_idle(s_empty + 8 * sc.s, sc.phase ^ 1));
                if (!ok) break;
                const uint32_t dst = s_ring + sc.s * WT_SCALE_BYTES + 2 * lane, zdst = z_ring + sc.s * WT_ZERO_BYTES + lane;
                // groups past the last and rows past the last get zeros: their weights are zeros
                // (every load of a batch is requested before the first is used: one round trip a batch, not one a load)
                if (by_four) {
                    for (int b = 0; b < per_block; b += 8) {      // item i: groups 4 (i / 4) .. + 3 of 32 rows
                        uint2 v[8];
#pragma unroll
                        for (int u = 0; u < 8; ++u) {
                            const int i = b + u, n = n0 + lane + 32 * (i & 3), jj = i & ~3;
                            v[u] = make_uint2(0, 0);
                            if (i < per_block && n < p.N && j0 + jj < j_end) v[u] = __ldg(reinterpret_cast<const uint2*>(p.scale + (size_t)n * p.J + j0 + jj));
                        }
#pragma unroll
                        for (int u = 0; u < 8; ++u) {
                            const int i = b + u;
                            if (i >= per_block) break;
                            const uint32_t d = dst + 2 * ((i & ~3) * 128 + 32 * (i & 3));
                            sts16(d, __float2half_rn(__uint_as_float(v[u].x << 16) * OPERAND_SCALE));
                            sts16(d + 256, __float2half_rn(__uint_as_float(v[u].x & 0xffff0000u) * OPERAND_SCALE));
                            sts16(d + 512, __float2half_rn(__uint_as_float(v[u].y << 16) * OPERAND_SCALE));
                            sts16(d + 768, __float2half_rn(__uint_as_float(v[u].y & 0xffff0000u) * OPERAND_SCALE));
                        }
                    }
                } else {
                    for (int b = 0; b < 4 * per_block; b += 16) {      // item i: group i / 4 of 32 rows
                        unsigned short v[16];
#pragma unroll
                        for (int u = 0; u < 16; ++u) {
                            const int i = b + u, n = n0 + lane + 32 * (i & 3), jj = i >> 2;
                            v[u] = n < p.N && j0 + jj < j_end ? __ldg(p.scale + (size_t)n * p.J + j0 + jj) : (unsigned short)0;
                        }
#pragma unroll
                        for (int u = 0; u < 16; ++u) {
                            const int i = b + u;
                            sts16(dst + 2 * ((i >> 2) * 128 + 32 * (i & 3)), __float2half_rn(bf16_bits_to_float(v[u]) * OPERAND_SCALE));
                        }
                    }
                }
                if (p.zero) {
                    for (int b = 0; b < 4 * per_block; b += 16) {
                        unsigned char v[16];
#pragma unroll
                        for (int u = 0; u < 16; ++u) {
                            const int i = b + u, n = n0 + lane + 32 * (i & 3), jj = i >> 2;
                            v[u] = n < p.N && j0 + jj < j_end ? __ldg(p.zero + (size_t)n * p.J + j0 + jj) : (unsigned char)0;
                        }
#pragma unroll
                        for (int u = 0; u < 16; ++u) {
                            const int i = b + u;
                            sts8(zdst + (i >> 2) * 128 + 32 * (i & 3), v[u]);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(s_full + 8 * sc.s);
                sc.next(WT_SS);
            }
        }
        if (!ok && lane == 0) atomicCAS(t.status, 0, 26);
    }
    // -------------------------------------------------------------------------------------------- epilogue
    // Four warps finish the tiles while the others work on the next one. At the last tile nothing is left to unpack, and the
    // warps that did so share in it: each set of four takes every fourth chunk of 16 rows of x (2048 x 1280 x 5120 with a
    // residual: 28.6 us without them, 24.7 us with them).
    if (warp < WT_X && ok && last >= 0 && (!SPLIT || warp >= WT_EPILOGUE)) {
        // SPLIT: this CTA's sums of the chunks that other ranks finish go to those; true once every rank has done so
        auto share_sums = [&](int rows, uint32_t tacc, int row) {
            const bool done = __all_sync(0xffffffffu, mbar_wait_idle(last_full, 0));
            fence_after_sync();
            cluster_wait();      // the other CTAs run
            if (done) {
                for (int i = 0; i * 16 < rows; ++i) {
                    const uint32_t owner = i % t.split, slot = i / t.split;
                    if (owner == part) continue;
                    uint32_t r[16];
                    tmem_ld_32x16(tacc + 16 * i, r);
                    tmem_ld_wait();
                    const uint32_t to = mapa_shared(sums + (slot * (t.split - 1) + part - ((int)owner < (int)part)) * 8192 + row * 4, owner);
#pragma unroll
                    for (int e = 0; e < 16; ++e) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to + e * 512), "r"(r[e]) : "memory");
                }
            }
            cluster_sync_all();
            return done;
        };
        Ring acc;
        if (warp < WT_EPILOGUE) acc.s = (last - item0) / item_stride % t.n_acc;
        for (int tile = warp < WT_EPILOGUE ? last : item0; tile <= last && ok; tile += item_stride) {
            const bool shared_tile = tile == last;
            const int set = shared_tile ? warp >> 2 : 0, sets = shared_tile ? WT_X / 4 : 1;
            const int quarter = warp & 3, row = quarter * 32 + lane;
            int m0, n0;
            rows_of(tile, m0, n0);
            const int n = n0 + row;
            const bool in = n < p.N;
            const float bias = p.bias && in ? __half2float(p.bias[n]) : 0.f;
            const uint32_t tacc = tmem_base + acc.s * t.acc_stride + ((uint32_t)(quarter * 32) << 16);
            const int rows = min(t.bt, p.M - m0);
            // A thread holds one column n of the result and consecutive rows m. Neighbouring threads swap halves so that the
            // even one has (n, n + 1) of row m and the odd one of row m + 1: a store covers two rows of 64 bytes. The options
            // are uniform and each is a loop of its own (as branches per element they took 84 cycles an element).
            const int np = n & ~1, mp = m0 + (lane & 1);
            const uint32_t mine = lane & 1 ? 0x3276u : 0x5410u;
            auto load_residual = [&](auto pairs, int c, uint32_t (&res)[8]) {
                const int left = rows - c;
                if constexpr (decltype(pairs)::value) {
                    const __half* src = p.residual + (long long)(mp + c) * p.ldr + np;
#pragma unroll
                    for (int i = 0; i < 8; ++i, src += 2 * p.ldr) {
                        res[i] = 0;
                        if (in && 2 * i + (lane & 1) < left) res[i] = *reinterpret_cast<const uint32_t*>(src);
                    }
                } else {
                    const unsigned short* src = reinterpret_cast<const unsigned short*>(p.residual) + (long long)(m0 + c) * p.ldr + n;
#pragma unroll
                    for (int i = 0; i < 8; ++i, src += 2 * p.ldr) {
                        res[i] = 0;
                        if (in && 2 * i < left) res[i] = src[0];
                        if (in && 2 * i + 1 < left) res[i] |= (uint32_t)src[p.ldr] << 16;
                    }
                }
            };
            if (p.residual && warp >= WT_EPILOGUE) {      // into L2 while the main loop runs: a lane asks for a row's 64 bytes of this warp
                const __half* line = p.residual + (long long)(m0 + lane) * p.ldr + n0 + quarter * 32;
                if (n0 + quarter * 32 < p.N)
                    for (int m = lane; m < rows; m += 32, line += 32 * p.ldr) asm volatile("prefetch.global.L2 [%0];" ::"l"(line));
            }
            auto store_tile = [&](auto pairs) {
                constexpr bool PAIRS = decltype(pairs)::value;
                const int first = 16 * (SPLIT ? (int)part : set), hop = 16 * (SPLIT ? t.split : sets);
                uint32_t res[8];      // the residual of the next 16 rows of x
                if (p.residual) load_residual(pairs, first, res);
                if constexpr (SPLIT) {
                    if (!share_sums(rows, tacc, row)) return false;
                } else {
                    if (!__all_sync(0xffffffffu, mbar_wait_idle(shared_tile ? last_full : acc_full + 8 * acc.s, shared_tile ? 0 : acc.phase))) return false;
                    fence_after_sync();
                }
                for (int c = first; c < rows; c += hop) {
                    uint32_t r[16];
                    tmem_ld_32x16(tacc + c, r);
                    tmem_ld_wait();
                    float v[16];
                    if constexpr (SPLIT) {
                        const uint32_t from = sums + (c / hop) * (t.split - 1) * 8192 + row * 4;
#pragma unroll
                        for (int e = 0; e < 16; ++e) v[e] = 0.f;
                        for (int s = 0; s < t.split; ++s) {      // in rank order, whichever rank adds
#pragma unroll
                            for (int e = 0; e < 16; ++e)
                                v[e] += s == (int)part ? __uint_as_float(r[e]) : lds_f32(from + (s - (s > (int)part)) * 8192 + e * 512);
                        }
#pragma unroll
                        for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(v[e]);
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) v[e] = fmaf(__uint_as_float(r[e]), OPERAND_UNSCALE, bias);
                    if (p.act == KATZ_ACT_SILU) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) v[e] = silu_f(v[e]);
                    }
                    if (p.residual) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            uint32_t w = res[i];
                            if (PAIRS) w = __byte_perm(w, __shfl_xor_sync(0xffffffffu, w, 1), mine);
                            const float2 f = unpack_half2(w);
                            v[2 * i] += f.x;
                            v[2 * i + 1] += f.y;
                        }
                        load_residual(pairs, c + hop, res);      // nothing past the last row
                    }
                    const int left = rows - c;
                    uint32_t o[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[i] = pack_half2(v[2 * i] * p.out_scale, v[2 * i + 1] * p.out_scale);
                    if constexpr (PAIRS) {
                        __half* dst = p.out + (long long)(mp + c) * p.ldo + np;
#pragma unroll
                        for (int i = 0; i < 8; ++i, dst += 2 * p.ldo) {
                            o[i] = __byte_perm(o[i], __shfl_xor_sync(0xffffffffu, o[i], 1), mine);
                            if (in && 2 * i + (lane & 1) < left) *reinterpret_cast<uint32_t*>(dst) = o[i];
                        }
                    } else {
                        unsigned short* dst = reinterpret_cast<unsigned short*>(p.out) + (long long)(m0 + c) * p.ldo + n;
#pragma unroll
                        for (int i = 0; i < 8; ++i, dst += 2 * p.ldo) {
                            if (in && 2 * i < left) dst[0] = (unsigned short)o[i];
                            if (in && 2 * i + 1 < left) dst[p.ldo] = (unsigned short)(o[i] >> 16);
                        }
                    }
                }
                return true;
            };
            ok = t.in_pairs ? store_tile(std::true_type{}) : store_tile(std::false_type{});
            if (shared_tile || !ok) break;
            fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                if (PAIR) mbar_arrive_cluster_tmem(mapa_shared(acc_empty + 8 * acc.s, 0));
                else mbar_arrive(acc_empty + 8 * acc.s);
            }
            acc.next(t.n_acc);
        }
        if (!ok && lane == 0) atomicCAS(t.status, 0, 22);
    }
    // -------------------------------------------------------------------------------------------- teardown
    __syncwarp();
    if (SPLIT && (warp < WT_EPILOGUE || warp >= WT_X)) {      // the epilogue warps' two barriers of share_sums()
        cluster_wait();
        cluster_sync_all();
    }
    fence_before_sync();
    __syncthreads();
    if (PAIR) cluster_sync_all();      // neither CTA leaves (or frees TMEM) while the other may still signal it or read its tiles
    if (warp == WT_MMA) {
        fence_after_sync();
        if (PAIR) tmem_dealloc_pair(tmem_base, WT_TMEM_COLS);
        else tmem_dealloc(tmem_base, WT_TMEM_COLS);
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn get_encode() {
    static const EncodeTiledFn fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult qres;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &qres) != cudaSuccess ||
            qres != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<EncodeTiledFn>(f);
    }();
    return fn;
}

static int encode_rows(CUtensorMap* map, CUtensorMapDataType type, CUtensorMapSwizzle swizzle, const void* base, uint64_t inner,
                       uint64_t outer, uint64_t row_bytes, uint32_t box_inner, uint32_t box_outer) {
    EncodeTiledFn enc = get_encode();
    if (!enc) return KATZ_ENOTREADY;
    cuuint64_t dims[2] = {inner, outer};
    cuuint64_t strides[1] = {row_bytes};
    cuuint32_t box[2] = {box_inner, box_outer};
    cuuint32_t es[2] = {1, 1};
    CUresult r = enc(map, type, 2, const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : KATZ_EINVAL;
}

struct W4Device {
    int slots[4];      // clusters of 1, 2, 4 and 8 CTAs that are resident at once
    bool ready;
};

static int device_limits(W4Device& out) {
    static W4Device cached[KATZ_MAX_DEVICES] = {};
    static std::mutex first_calls;      // callers' threads hold no lock of ours
    std::lock_guard<std::mutex> lock(first_calls);
    W4Device& d = cached[current_device_index()];
    if (!d.ready) {
        W4Device found{};
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&found.slots[0], cudaDevAttrMultiProcessorCount, dev);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(linear_w4_tc05_kernel<false, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, WT_MAX_SMEM);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(linear_w4_tc05_kernel<true, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, WT_MAX_SMEM);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(linear_w4_tc05_kernel<false, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, WT_MAX_SMEM);
        for (int i = 1; e == cudaSuccess && i < 4; ++i) {
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3((found.slots[0] >> i) << i);
            cfg.blockDim = dim3(WT_THREADS);
            cfg.dynamicSmemBytes = WT_MAX_SMEM;
            cudaLaunchAttribute at[1];
            at[0].id = cudaLaunchAttributeClusterDimension;
            at[0].val.clusterDim.x = 1 << i;
            at[0].val.clusterDim.y = 1;
            at[0].val.clusterDim.z = 1;
            cfg.attrs = at;
            cfg.numAttrs = 1;
            e = i == 1 ? cudaOccupancyMaxActiveClusters(&found.slots[i], linear_w4_tc05_kernel<true, false>, &cfg)
                       : cudaOccupancyMaxActiveClusters(&found.slots[i], linear_w4_tc05_kernel<false, true>, &cfg);
        }
        if (e != cudaSuccess) return (int)e;
        found.ready = true;
        d = found;
    }
    out = d;
    return 0;
}

// bytes of the other ranks' sums that a CTA receives
static int sums_bytes(int bt, int split) { return (split - 1) * ceil_div(ceil_div(bt, 16), split) * 8192; }

int linear_w4_tc05(const W4Params& p, cudaStream_t st) {
    W4Device dev;
    int rc = device_limits(dev);
    if (rc) return rc;
    // Tile choice: the least modelled time (cycles) over the number of tiles along M: single CTAs, pairs, or clusters that
    // split K. Per unit of 128 k a single CTA spends 4 BT cycles in the tensor pipe, its loads at about 48 bytes a cycle from
    // L2, and 660 cycles of unpacking (measured: 0.35 us a unit at BT 80, 0.42 at 128, 0.5 at 160); a pair 5.6 BT, at least 820
    // (0.43 us at 96, 0.5 at 160, 0.6 at 192, 0.75 at 240, all SMs at work and the clock down with them). Between tiles and
    // after the last one the epilogue, which all warps share at the end. 2048 x 8192 x 8192: pairs of BT 128 218 us, 160 196 us,
    // 240 189 us, 256 (a last wave half empty) 218 us; 512 x 8192 x 8192: 128 59 us, 256 51 us.
    const int units = ceil_div(p.K, 128);
    W4Tile t{};
    bool pair = false;
    double best = 1e30;
    const int min_tiles = ceil_div(p.M, p.N <= 128 ? 192 : 256);      // up to 128 weight rows are no pair's
    for (int mt = min_tiles; mt <= min_tiles + 8; ++mt) {
        const int bt = ceil_div(ceil_div(p.M, mt), 16) * 16, m_tiles = ceil_div(p.M, bt);
        for (int mode = -1; mode < 4; ++mode) {      // -1: pairs; i: K split over 2^i CTAs
            const bool two = mode < 0;
            const int split = two ? 1 : 1 << mode, n_tiles = ceil_div(p.N, two ? 256 : 128);
            const long long tiles = (long long)m_tiles * n_tiles;
            if (two ? p.N <= 128 : bt > 192) continue;      // a lone CTA has room for two stages of wider x only
            const int slots = dev.slots[two ? 1 : mode];
            if (slots < 1 || (split > 1 && (tiles > slots || units < 2 * split))) continue;
            const int x_bytes = bt * (two ? 128 : 256);
            if ((WT_MAX_SMEM - WT_FIXED_SMEM - sums_bytes(bt, split)) / x_bytes < 2) continue;
            const int n_acc = bt <= 160 && tiles > slots ? 2 : 1;      // three stages of 64 columns beside two accumulators
            const double waves = (double)ceil_div_ll(tiles, slots), drain = 600.0 + 8.0 * bt;
            const double unit = std::max(std::max(two ? 5.6 * bt : 4.0 * bt, (x_bytes + 8192.0) / 48.0), two ? 820.0 : 660.0);
            const double cost = waves * ceil_div(units, split) * unit + (waves - 1.0) * (n_acc == 1 ? drain : 100.0) + (split > 1 ? drain + 3000.0 : 600.0 + 2.5 * bt);
            if (cost < best) {
                best = cost;
                pair = two;
                t.bt = bt;
                t.m_tiles = m_tiles;
                t.n_tiles = n_tiles;
                t.n_acc = n_acc;
                t.split = split;
                t.x_bytes = x_bytes;
            }
        }
    }
    KATZ_CHECK_ARG(best < 1e30 && (long long)t.m_tiles * t.n_tiles < (1ll << 28), KATZ_ESIZE);
    t.acc_stride = ceil_div(t.bt, 32) * 32;
    const int fixed = WT_FIXED_SMEM + sums_bytes(t.bt, t.split);
    t.x_stages = std::min((WT_MAX_SMEM - fixed) / t.x_bytes, WT_XS);
    t.a_stages = std::min((WT_TMEM_COLS - t.n_acc * t.acc_stride) / 64, WT_AS);
    KATZ_CHECK_ARG(t.a_stages >= WT_GROUPS && t.x_stages >= 2, KATZ_ESIZE);      // holds for every tile the choice above makes
    t.in_pairs = ((p.N | p.ldo) & 1) == 0 && ((uintptr_t)p.out & 3) == 0 &&
                 (!p.residual || ((p.ldr & 1) == 0 && ((uintptr_t)p.residual & 3) == 0));
    t.status = tc05_status_device_ptr();
    if (!t.status) return KATZ_ENOTREADY;
    CUtensorMap tx, tq;
    rc = encode_rows(&tx, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, CU_TENSOR_MAP_SWIZZLE_128B, p.x, p.K, p.M, (uint64_t)p.ldx * 2, 64,
                     pair ? t.bt / 2 : t.bt);
    if (rc) return rc;
    rc = encode_rows(&tq, CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_64B, p.q, p.K / 2, p.N, p.K / 2, 64, 128);
    if (rc) return rc;
    const int smem = t.x_stages * t.x_bytes + fixed, tiles = t.m_tiles * t.n_tiles;
    if (t.split > 1) launch_k_cluster(linear_w4_tc05_kernel<false, true>, tiles * t.split, WT_THREADS, smem, st, t.split, tx, tq, p, t);
    else if (pair) launch_k_cluster(linear_w4_tc05_kernel<true, false>, 2 * std::min(tiles, dev.slots[1]), WT_THREADS, smem, st, 2, tx, tq, p, t);
    else launch_k_cluster(linear_w4_tc05_kernel<false, false>, std::min(tiles, dev.slots[0]), WT_THREADS, smem, st, 1, tx, tq, p, t);
    KATZ_LAUNCH_RET();
}

}  // namespace katz
