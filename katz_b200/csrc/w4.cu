// 4-bit weights with group scales (w4.cuh has the format): made from fp16 weights, read back, and multiplied with few rows.
#include <algorithm>

#include "tc05.cuh"      // packed fp32 arithmetic
#include "w4.cuh"
#include "katz_b200.h"

namespace katz {

using namespace w4;

// ---------------------------------------------------------------------------------------------------------------------
// fp16 -> codes and scales. Per group: scale = bf16(max |w| / 7), code = 8 + rint(w / scale) with ties to even. The quotient
// is the correctly rounded one (a product with the reciprocal and Markstein's residual correction): w and scale have 11 and 8 significant
// bits, so a quotient that is not exactly half way between two codes is at least 2^-13 of its size away from there, and one
// that is comes out exact. |w / scale| <= 7 * (1 + 2^-8): no code leaves 1..15.
// A group that holds an infinity or a NaN gets a NaN scale: what is read back of it is NaN, never a plausible number.
//
// Bound by HBM (2.5 bytes per weight and the scales), which leaves about ten instructions a weight. A lane holds 8 weights; a
// group is 4, 8 or 16 neighbouring lanes; a warp works on W4_PIECES pieces of 256 weights so that enough loads are in flight.
// FLAT (contiguous rows of whole groups): the matrix is one run of groups and no lane is idle at a row's end.
// 166400 x 2048, quantised and read back: 264 us for 1725 MB, HBM's copy rate (6.54 TB/s); 1280 x 1280: 3.7 us, two launches.
constexpr int W4_PIECES = 4;

__device__ __forceinline__ __half2 hmax2_abs_nan(__half2 a, __half2 b) { return __hmax2_nan(__habs2(a), __habs2(b)); }

// piece i of this warp: the row and k of this lane's 8 weights (FLAT: row 0, k over the whole matrix)
template <bool FLAT>
struct Piece {
    long long row, k;
    bool in;
    __device__ __forceinline__ Piece(uint32_t index, uint32_t total, uint32_t pieces_per_row, long long K, int lane) {
        row = FLAT ? 0 : index / pieces_per_row;
        k = (long long)(FLAT ? index : index - (uint32_t)row * pieces_per_row) * 256 + lane * 8;
        in = index < total && k < K;
    }
};

template <int GROUP, bool FLAT>
__global__ void __launch_bounds__(256) quantize_w4_kernel(const __half* __restrict__ w, long long ldw, unsigned char* __restrict__ q,
                                                          unsigned short* __restrict__ scale, long long K, int J, uint32_t total,
                                                          uint32_t pieces_per_row) {
    pdl_wait();      // writes weights: the next kernel is not released early
    constexpr int LANES = GROUP / 8;
    const int lane = threadIdx.x & 31;
    const uint32_t first = (blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * W4_PIECES;
    uint4 v[W4_PIECES];
#pragma unroll
    for (int i = 0; i < W4_PIECES; ++i) {
        const Piece<FLAT> at(first + i, total, pieces_per_row, K, lane);
        v[i] = make_uint4(0, 0, 0, 0);
        if (at.in) v[i] = __ldg(reinterpret_cast<const uint4*>(w + at.row * ldw + at.k));
    }
#pragma unroll
    for (int i = 0; i < W4_PIECES; ++i) {
        if (first + i >= total) return;      // uniform over the warp
        const uint32_t u[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
        __half2 m2 = hmax2_abs_nan(hmax2_abs_nan(as_half2(u[0]), as_half2(u[1])), hmax2_abs_nan(as_half2(u[2]), as_half2(u[3])));
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) m2 = hmax2_abs_nan(m2, as_half2(__shfl_xor_sync(0xffffffffu, as_u32(m2), o)));
        const float top = __half2float(__hmax_nan(__low2half(m2), __high2half(m2)));
        // top / 7 rounded once (a product and one residual step), then to bf16: 11 bits over 7 are never so near the middle of
        // two bf16 numbers that the first rounding decides, unless they are exactly there
        float s7 = top * (1.0f / 7.0f);
        s7 = fmaf(fmaf(-7.0f, s7, top), 1.0f / 7.0f, s7);
        __nv_bfloat16 sb = __float2bfloat16_rn(s7);
        if (!(top <= 65504.0f)) sb = __float2bfloat16_rn(__uint_as_float(0x7fc00000u));
        const float s = __bfloat162float(sb);
        float inv;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
        if (!(s > 0.f)) inv = 0.f;
        const float2 inv2 = make_float2(inv, inv), s2 = make_float2(-s, -s), magic = make_float2(12582912.0f, 12582912.0f);
        // Adding 1.5 * 2^23 rounds to an integer n (ties to even) and leaves 0x4b400000 + n as the float's bits. Summed with
        // weights 16^e they are the eight n in base 16, plus a constant; 8 is the code of zero.
        uint32_t codes = 0x88888888u - 0x4b400000u * 0x11111111u;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 f = unpack_half2(u[e]);
            float2 t = tc05::mul2(f, inv2);
            t = tc05::fma2(tc05::fma2(t, s2, f), inv2, t);
            t = tc05::add2(t, magic);
            codes += (__float_as_uint(t.x) << (8 * e)) + (__float_as_uint(t.y) << (8 * e + 4));
        }
        const Piece<FLAT> at(first + i, total, pieces_per_row, K, lane);
        if (at.in) {
            *reinterpret_cast<uint32_t*>(q + at.row * (K / 2) + at.k / 2) = codes;
            if ((lane & (LANES - 1)) == 0) scale[at.row * J + at.k / GROUP] = __bfloat16_as_ushort(sb);
        }
    }
}

// codes, scales -> fp16(scale * (code - zero)), one rounding. Bound by HBM (2.5 bytes per weight); the same shape as above.
template <int GROUP, bool FLAT>
__global__ void __launch_bounds__(256) dequantize_w4_kernel(const unsigned char* __restrict__ q, const unsigned short* __restrict__ scale,
                                                            const unsigned char* __restrict__ zero, __half* __restrict__ w,
                                                            long long ldw, long long K, int J, uint32_t total, uint32_t pieces_per_row) {
    pdl_wait();      // writes weights: the next kernel is not released early
    const int lane = threadIdx.x & 31;
    const uint32_t first = (blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * W4_PIECES;
    uint32_t v[W4_PIECES];
    unsigned short sb[W4_PIECES];
    unsigned char zb[W4_PIECES];
#pragma unroll
    for (int i = 0; i < W4_PIECES; ++i) {
        const Piece<FLAT> at(first + i, total, pieces_per_row, K, lane);
        v[i] = 0;
        sb[i] = 0;
        zb[i] = 8;
        if (at.in) {
            const long long j = at.row * J + at.k / GROUP;
            v[i] = __ldg(reinterpret_cast<const uint32_t*>(q + at.row * (K / 2) + at.k / 2));
            sb[i] = __ldg(scale + j);
            if (zero) zb[i] = __ldg(zero + j);
        }
    }
#pragma unroll
    for (int i = 0; i < W4_PIECES; ++i) {
        const Piece<FLAT> at(first + i, total, pieces_per_row, K, lane);
        if (!at.in) continue;
        __half2 d[4];
        unpack8(v[i], as_half2(0xe400e400u + zb[i] * 0x00010001u), as_half2(0xd400d400u + zb[i] * 0x00100010u), d);
        const float s = bf16_bits_to_float(sb[i]);
        float2 f[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = tc05::mul2(__half22float2(d[e]), make_float2(s, s));
        *reinterpret_cast<uint4*>(w + at.row * ldw + at.k) = make_uint4(pack_half2(f[0].x, f[1].x), pack_half2(f[2].x, f[3].x),
                                                                        pack_half2(f[0].y, f[1].y), pack_half2(f[2].y, f[3].y));
    }
}

struct PieceGrid {
    long long K;             // of a row, FLAT: of the matrix
    uint32_t total, per_row, ctas;
    bool flat, ok;
};
static PieceGrid piece_grid(int N, int K, int group, long long ldw) {
    PieceGrid g{};
    g.flat = (ldw == K || N == 1) && K % group == 0;
    g.K = g.flat ? (long long)N * K : K;
    const long long per_row = ceil_div_ll(g.K, 256), total = g.flat ? per_row : N * per_row;
    g.per_row = (uint32_t)per_row;
    g.total = (uint32_t)total;
    g.ctas = (uint32_t)ceil_div_ll(total, 8 * W4_PIECES);
    g.ok = total < (1ll << 31);
    return g;
}

// ---------------------------------------------------------------------------------------------------------------------
// Few rows: out[M, N] = (act(x W^T + bias) + residual) * out_scale with W in 4 bits.
//
// Sixteen weight rows are the M side of m16n8k16 products, up to eight rows of x the N side. Lane (g = lane / 4, t = lane % 4)
// holds the codes of weight rows g and g + 8 over 32 consecutive k (16 bytes of each, inside one group whatever its size) as
// four words of eight k; a word of each row makes the A operands of two products. The sum over k may be taken in any order as
// long as both operands use the same one, so the codes are used as they lie in memory, and x is put into the order that the
// unpacking gives, pairs (k, k + 4). The warps of a CTA take turns over blocks of 128 k; their sums meet in shared memory, added
// in warp order. Two kernels differ in how the data reaches the lanes:
//
// direct: each lane loads what it needs when it needs it, a CTA for every 16 weight rows. Nothing to set up, but a block's
// latency stands between two blocks of a warp, and x is fetched again by every CTA. Right for weights whose whole reduction is
// in flight at once. 1 x 1280 x 1280: 2.3 us (streamed 3.1), 1 x 13760 x 1280: 5.6 us (6.3), 8 x 13760 x 1280: 6.0 us (8.5).
//
// stream: persistent CTAs, as many as fit, hold x in shared memory, 16 bytes a lane and word, no two lanes in one bank. Each
// warp streams its codes through a ring in shared memory with asynchronous copies, across row tiles, every lane reading back
// what it copied itself: HBM's latency needs some 45 KB in flight an SM. Scales and zero points of a tile lie in shared memory,
// copied row by row while the tile before is multiplied. 1 x 5120 x 5120: 9.0 us (direct 11.2), 1 x 16384 x 8192 with groups of
// 128: 20 us (direct 31; the codes alone at HBM's rate: 10), 1 x 32768 x 8192: 32 us (direct 59). Above HBM's rate it is bound
// by instructions: some 200 a block and warp (72 turn codes into operands, 8 multiply), the issue slots 64% busy, DRAM 34%.
// Where the group is a block (128), the products take the integers code - zero and the scale multiplies their fp32 sum;
// smaller groups differ from lane to lane, and the scale multiplies the operand (w4.cuh; on the whole block it costs 10% more).
// (x is rows, N, K here; weights larger than L2, groups of 64 where none are named.)
constexpr int W4_ROWS_THREADS = 512;
constexpr int W4_RING = 4;                    // blocks of a warp in flight or in use

// 16 bytes of codes, global -> shared, zeros if !in. L2 fetches the 256 bytes around them, most of which the CTA's
// other warps are about to ask for: a row at a time a warp reads 64 bytes, and HBM gives such pieces at half its rate.
__device__ __forceinline__ void copy_codes(uint32_t dst, const unsigned char* src, bool in) {
    asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}

// stride of a row of scales in shared memory: an odd number of 4-byte words, so that eight rows lie in different banks
static __host__ __device__ inline int scale_stride(int J) { return (J + 1) / 2 % 2 ? (J + 1) / 2 * 2 : (J + 1) / 2 * 2 + 2; }
// bytes of a row of x in shared memory: neighbouring rows 64 bytes apart modulo 128
static __host__ __device__ inline int x_row_bytes(int K) { return (K + 127) / 128 * 256 + 64; }

// eight values of x as the pairs (0,4), (1,5), (2,6), (3,7)
__device__ __forceinline__ uint4 load_x_pairs(const __half* src, bool aligned) {
    uint4 v;
    if (aligned) {
        v = *reinterpret_cast<const uint4*>(src);
    } else {
        const unsigned short* e = reinterpret_cast<const unsigned short*>(src);
        v = make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16, e[6] | (uint32_t)e[7] << 16);
    }
    return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                      __byte_perm(v.y, v.w, 0x7632));
}

// One warp's stream of codes: of row tiles blockIdx.x, + gridDim.x, ... the blocks warp, + warps, ... of 128 k, through W4_RING
// slots of 1 KB in shared memory. A lane copies, and reads back, its words of weight rows g and g + 8.
struct CodeStream {
    const W4Params& p;
    const int blocks, tiles, warps, warp, hop, g, t;
    const uint32_t at;      // this lane's place in slot 0
    int tile, kb;           // the next block to copy
    uint32_t write_slot = 0, read_slot = 0;
    const unsigned char* src[2];      // this lane's codes of it

    // warps_ of the CTA's share a tile, this is warp_ of them; hop_: from this warp's tile to its next
    __device__ __forceinline__ CodeStream(const W4Params& p_, uint32_t ring, int warps_, int warp_, int tile_, int hop_)
        : p(p_), blocks((p_.K + 127) / 128), tiles((p_.N + 15) / 16), warps(warps_), warp(warp_), hop(hop_), g((threadIdx.x & 31) >> 2),
          t(threadIdx.x & 3), at(ring + (threadIdx.x >> 5) * W4_RING * 1024 + (threadIdx.x & 31) * 16), tile(tile_), kb(warp_) {
        at_tile();
    }
    __device__ __forceinline__ void at_tile() {
#pragma unroll
        for (int h = 0; h < 2; ++h)      // rows past the last are computed and not stored
            src[h] = p.q + (size_t)min(tile * 16 + 8 * h + g, p.N - 1) * (p.K / 2) + warp * 64 + 16 * t;
    }
    __device__ __forceinline__ void copy_next() {
        if (tile < tiles) {
            // K is a multiple of 32: a lane's codes exist together or not at all (only the last block lacks any)
            const bool in = kb * 128 + 32 * t < p.K;
#pragma unroll
            for (int h = 0; h < 2; ++h) copy_codes(at + write_slot + h * 512, in ? src[h] : p.q, in);
            kb += warps;
            src[0] += warps * 64;
            src[1] += warps * 64;
            if (kb >= blocks) {
                kb = warp;
                tile += hop;
                at_tile();
            }
        }
        cp_async_commit();
        write_slot = (write_slot + 1024) % (W4_RING * 1024);
    }
    __device__ __forceinline__ void start() {
#pragma unroll
        for (int i = 0; i < W4_RING - 1; ++i) copy_next();
    }
    // the next block's words; requests one more, into the slot that was read in the round before
    __device__ __forceinline__ void next(uint32_t (&v)[2][4]) {
        cp_async_wait<W4_RING - 2>();
        const uint4 a = lds128(at + read_slot), b = lds128(at + read_slot + 512);
        read_slot = (read_slot + 1024) % (W4_RING * 1024);
        copy_next();
        v[0][0] = a.x, v[0][1] = a.y, v[0][2] = a.z, v[0][3] = a.w;
        v[1][0] = b.x, v[1][1] = b.y, v[1][2] = b.z, v[1][3] = b.w;
    }
};

// Scales and zero points of the tiles' rows in shared memory, a buffer of 16 rows a tile. They are copied asynchronously, with
// the codes of the first block of the tile `ahead` tiles earlier: by that tile's successors' last waits the copy is over
// (ahead * blocks of a warp >= W4_RING - 1), and the barrier at a tile's end shows it to the other warps. Rows that do not
// start on 4-byte boundaries (J odd; zero points: J % 4) are loaded and stored.
struct ScaleRows {
    int ahead, sld, zld;      // strides of a row of scales (elements) and of zero points (bytes)
    bool async_scale, async_zero;
};
static ScaleRows scale_rows(const W4Params& p, int warps) {
    ScaleRows s;
    const int blocks = ceil_div(p.K, 128), least = blocks / warps;      // blocks of the warp that has fewest
    s.ahead = ceil_div(W4_RING - 1, least > 0 ? least : 1);
    s.sld = scale_stride(p.J);
    s.zld = ceil_div(p.J, 4) * 4 + 4;
    s.async_scale = p.J % 2 == 0 && ((uintptr_t)p.scale & 3) == 0;
    s.async_zero = p.J % 4 == 0 && ((uintptr_t)p.zero & 3) == 0;
    return s;
}
static long long scale_rows_bytes(const W4Params& p, int warps, int teams) {
    const ScaleRows s = scale_rows(p, warps);
    return (s.ahead + 1ll) * 16 * teams * (s.sld * 2 + (p.zero ? s.zld : 0));
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
template <bool ZERO, int ROWS>
__device__ __forceinline__ void read_scales(const W4Params& p, const ScaleRows& s, int n0, unsigned short* scales, unsigned char* zeros) {
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    for (int r = threadIdx.x >> 5; r < ROWS; r += warps) {
        const size_t at = (size_t)min(n0 + r, p.N - 1) * p.J;
        if (s.async_scale) {
            for (int j = 2 * lane; j < p.J; j += 64) copy4(smem_u32(scales + r * s.sld + j), p.scale + at + j);
        } else {
            for (int j = lane; j < p.J; j += 32) scales[r * s.sld + j] = __ldg(p.scale + at + j);
        }
        if (ZERO) {
            if (s.async_zero) {
                for (int j = 4 * lane; j < p.J; j += 128) copy4(smem_u32(zeros + r * s.zld + j), p.zero + at + j);
            } else {
                for (int j = lane; j < p.J; j += 32) zeros[r * s.zld + j] = __ldg(p.zero + at + j);
            }
        }
    }
}

__device__ __forceinline__ void finish(const W4Params& p, float v, long long m, int n) {
    if (p.bias) v += __half2float(p.bias[n]);
    if (p.act == KATZ_ACT_SILU) v = silu_f(v);
    if (p.residual) v += __half2float(p.residual[m * p.ldr + n]);
    p.out[m * p.ldo + n] = __float2half_rn(v * p.out_scale);
}

// Any M (8 * MT rows a CTA) and any alignment of x.
template <int MT, bool XALIGNED>
__global__ void __launch_bounds__(W4_ROWS_THREADS) linear_w4_direct_kernel(const __grid_constant__ W4Params p) {
    __shared__ float red[W4_ROWS_THREADS / 32][8 * MT][16 + 4];
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int tiles = (p.N + 15) / 16, n0 = blockIdx.x % tiles * 16, m0 = blockIdx.x / tiles * 8 * MT, blocks = (p.K + 127) / 128;
    float acc[MT][2][4] = {};      // two chains of products
    pdl_wait();
    pdl_launch_dependents();
    for (int kb = warp; kb < blocks; kb += warps) {
        const int k = kb * 128 + 32 * t;
        const bool in = k < p.K;      // K is a multiple of 32: a lane's 32 k exist together or not at all
        uint32_t v[2][4];
        __half2 scale[2], low[2], high[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int n = min(n0 + 8 * h + g, p.N - 1);      // rows past the last are computed and not stored
            const size_t j = (size_t)n * p.J + (k >> p.group_shift);
            uint4 w = make_uint4(0, 0, 0, 0);
            unsigned short sb = 0;
            uint32_t z = 8;
            if (in) {
                w = __ldg(reinterpret_cast<const uint4*>(p.q + (size_t)n * (p.K / 2) + k / 2));
                sb = __ldg(p.scale + j);
                if (p.zero) z = __ldg(p.zero + j);
            }
            v[h][0] = w.x, v[h][1] = w.y, v[h][2] = w.z, v[h][3] = w.w;
            scale[h] = __float2half2_rn(bf16_bits_to_float(sb) * OPERAND_SCALE);
            low[h] = as_half2(0xe400e400u + z * 0x00010001u);       // -(1024 + zero)
            high[h] = as_half2(0xd400d400u + z * 0x00100010u);      // -(64 + zero)
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint4 b[MT];
#pragma unroll
            for (int c = 0; c < MT; ++c) {
                const int m = m0 + 8 * c + g;
                b[c] = make_uint4(0, 0, 0, 0);
                if (in && m < p.M) b[c] = load_x_pairs(p.x + m * p.ldx + k + 8 * i, XALIGNED);
            }
            __half2 d[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                unpack8(v[h][i], low[h], high[h], d[h]);
#pragma unroll
                for (int e = 0; e < 4; ++e) d[h][e] = __hmul2(d[h][e], scale[h]);
            }
            const uint32_t a0[4] = {as_u32(d[0][0]), as_u32(d[1][0]), as_u32(d[0][1]), as_u32(d[1][1])};
            const uint32_t a1[4] = {as_u32(d[0][2]), as_u32(d[1][2]), as_u32(d[0][3]), as_u32(d[1][3])};
#pragma unroll
            for (int c = 0; c < MT; ++c) {
                const uint32_t b0[2] = {b[c].x, b[c].y}, b1[2] = {b[c].z, b[c].w};
                mma_f16_16816(acc[c][0], a0, b0);
                mma_f16_16816(acc[c][1], a1, b1);
            }
        }
    }
#pragma unroll
    for (int c = 0; c < MT; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[warp][8 * c + 2 * t + (e & 1)][g + 8 * (e >> 1)] = acc[c][0][e] + acc[c][1][e];
    __syncthreads();
    for (int i = threadIdx.x; i < 8 * MT * 16; i += blockDim.x) {
        const int ml = i / 16, nl = i % 16, n = n0 + nl;
        const long long m = m0 + ml;
        if (m >= p.M || n >= p.N) continue;
        float v = 0.f;
        for (int w = 0; w < warps; ++w) v += red[w][ml][nl];
        finish(p, v * OPERAND_UNSCALE, m, n);
    }
}

template <bool WIDE, bool ZERO, int TEAMS>
__global__ void __launch_bounds__(W4_ROWS_THREADS) linear_w4_stream_kernel(const __grid_constant__ W4Params p, const ScaleRows sr, bool xaligned) {
    extern __shared__ __align__(16) unsigned char rows_smem[];
    constexpr int LD = 16 + 4, ROWS = 16 * TEAMS;
    const int all = blockDim.x >> 5, self = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int warps = all / TEAMS, team = TEAMS > 1 && self >= warps ? 1 : 0, warp = self - team * warps;      // of the tile's
    const int hop = gridDim.x * TEAMS;
    const int sld = sr.sld, blocks = (p.K + 127) / 128, xld = x_row_bytes(p.K), tiles = (p.N + 15) / 16;
    unsigned char* xs = rows_smem;                                                        // [M][xld]
    unsigned char* ring = xs + p.M * xld;                                                 // [warp][W4_RING][2 rows][lane][16 bytes]
    float* red = reinterpret_cast<float*>(ring + all * W4_RING * 1024);                 // [warp][8][LD]
    unsigned short* scales = reinterpret_cast<unsigned short*>(red + all * 8 * LD);      // [ahead + 1][rows][sld]
    unsigned char* zeros = reinterpret_cast<unsigned char*>(scales + (sr.ahead + 1) * ROWS * sld);      // [ahead + 1][rows][zld]
    CodeStream codes(p, smem_u32(ring), warps, warp, blockIdx.x * TEAMS + team, hop);
    pdl_wait();
    pdl_launch_dependents();
    for (int a = 0; a < sr.ahead; ++a)
        if ((int)blockIdx.x * TEAMS + a * hop < tiles)
            read_scales<ZERO, ROWS>(p, sr, (blockIdx.x * TEAMS + a * hop) * 16, scales + a * ROWS * sld, zeros + a * ROWS * sr.zld);
    cp_async_commit();
    codes.start();
    for (int v = threadIdx.x; v < blocks * 16; v += blockDim.x) {
        const int k = v * 8;
        for (int m = 0; m < p.M; ++m)
            *reinterpret_cast<uint4*>(xs + m * xld + (k / 128 * 16 + k / 8 % 4 * 4 + k / 32 % 4) * 16) =
                k < p.K ? load_x_pairs(p.x + m * p.ldx + k, xaligned) : make_uint4(0, 0, 0, 0);
    }
    cp_async_wait<W4_RING - 1>();      // the first tiles' scales
    __syncthreads();
    // columns of x past the last row hold another row: what they give is not stored
    const uint32_t x_row = smem_u32(xs) + 16 * t + min(g, p.M - 1) * xld;
    int buf = 0;
    for (int tile = blockIdx.x * TEAMS; tile < tiles; tile += hop, buf = buf == sr.ahead ? 0 : buf + 1) {      // the first team's
        const long long later = (long long)tile + (long long)sr.ahead * hop;
        const int into = buf == 0 ? sr.ahead : buf - 1;      // the buffer that the tile before has left
        if (later < tiles) read_scales<ZERO, ROWS>(p, sr, (int)later * 16, scales + into * ROWS * sld, zeros + into * ROWS * sr.zld);
        const unsigned short* s_row = scales + (buf * ROWS + team * 16 + g) * sld;
        const unsigned char* z_row = zeros + (buf * ROWS + team * 16 + g) * sr.zld;
        float acc[2][4] = {};      // two chains of products
        for (int kb = tile + team < tiles ? warp : blocks; kb < blocks; kb += warps) {
            uint32_t v[2][4];
            codes.next(v);
            const int j = min((kb * 128 + 32 * t) >> p.group_shift, p.J - 1);      // past the last k x is zero
            __half2 low[2], high[2], scale[2];
            float wide[2], part[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                low[h] = as_half2(0xe408e408u);       // -(1024 + 8)
                high[h] = as_half2(0xd480d480u);      // -(64 + 8)
                if (ZERO) {
                    const uint32_t z = z_row[8 * h * sr.zld + j];
                    low[h] = as_half2(0xe400e400u + z * 0x00010001u);
                    high[h] = as_half2(0xd400d400u + z * 0x00100010u);
                }
                wide[h] = bf16_bits_to_float(s_row[8 * h * sld + j]);
                scale[h] = __float2half2_rn(kb * 128 + 32 * t < p.K ? wide[h] * OPERAND_SCALE : 0.f);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                __half2 d[2][4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    unpack8(v[h][i], low[h], high[h], d[h]);
                    if (!WIDE)
#pragma unroll
                        for (int e = 0; e < 4; ++e) d[h][e] = __hmul2(d[h][e], scale[h]);
                }
                const uint32_t a0[4] = {as_u32(d[0][0]), as_u32(d[1][0]), as_u32(d[0][1]), as_u32(d[1][1])};
                const uint32_t a1[4] = {as_u32(d[0][2]), as_u32(d[1][2]), as_u32(d[0][3]), as_u32(d[1][3])};
                const uint4 b = lds128(x_row + (kb * 4 + i) * 64);
                const uint32_t b0[2] = {b.x, b.y}, b1[2] = {b.z, b.w};
                if (WIDE && i == 0) {
                    mma_f16_16816_first(part[0], a0, b0);
                    mma_f16_16816_first(part[1], a1, b1);
                } else {
                    mma_f16_16816(WIDE ? part[0] : acc[0], a0, b0);
                    mma_f16_16816(WIDE ? part[1] : acc[1], a1, b1);
                }
            }
            if (WIDE)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[0][e] = fmaf(wide[e >> 1], part[0][e] + part[1][e], acc[0][e]);
        }
        cp_async_wait<W4_RING - 2>();      // the next tile's scales (and the next block)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[(self * 8 + 2 * t + (e & 1)) * LD + g + 8 * (e >> 1)] = acc[0][e] + acc[1][e];
        __syncthreads();
        for (int i = threadIdx.x; i < p.M * ROWS; i += blockDim.x) {
            const int m = i / ROWS, r = i - m * ROWS, of = r >> 4, nl = r & 15, n = tile * 16 + r;
            if (n >= p.N) continue;
            float v = 0.f;
            for (int w = 0; w < warps; ++w) v += red[((of * warps + w) * 8 + m) * LD + nl];
            finish(p, WIDE ? v : v * OPERAND_UNSCALE, m, n);
        }
        __syncthreads();
    }
    cp_async_wait<0>();
}

static int sm_count() {
    static int n[KATZ_MAX_DEVICES] = {};
    int& c = n[current_device_index()];
    if (!c) {
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&c, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || c <= 0) c = 148;
    }
    return c;
}

template <int MT>
static int launch_direct(const W4Params& p, bool xaligned, cudaStream_t st) {
    const int blocks = ceil_div(p.K, 128);
    const long long grid = (long long)ceil_div(p.N, 16) * ceil_div(p.M, 8 * MT);
    KATZ_CHECK_ARG(grid <= 0x7fffffff, KATZ_ESIZE);
    // as many warps as share the blocks of k evenly: eight, sixteen where the CTAs do not fill the SMs
    const int most = grid < sm_count() ? 16 : 8, warps = ceil_div(blocks, ceil_div(blocks, most));
    launch_k(xaligned ? linear_w4_direct_kernel<MT, true> : linear_w4_direct_kernel<MT, false>, (unsigned)grid, warps * 32, 0, st, p);
    KATZ_LAUNCH_RET();
}

// shared memory of a CTA of the streaming kernel: `teams` tiles at a time, `warps` on each
static long long stream_smem(const W4Params& p, int warps, int teams) {
    return (long long)p.M * x_row_bytes(p.K) + (long long)warps * teams * (W4_RING * 1024 + 8 * 20 * 4) + scale_rows_bytes(p, warps, teams);
}
struct StreamPlan {
    int warps, teams;      // 0 warps: x and the scales do not fit
};
// Warps of a tile: as many as share its blocks of k evenly, up to eight or sixteen; what a tile costs outside its blocks
// (barriers, sums) is spread over twice as many of them with eight. Eight where four such CTAs fit an SM. With more x in shared
// memory two tiles of eight warps at a time, unless the SM with most work gets more tiles that way (1 x 32768 x 8192, groups of 128:
// 14 tiles either way, 36.3 -> 32.3 us; 1 x 16384 x 8192: 8 tiles instead of 7, 20.1 -> 20.8), then sixteen.
static StreamPlan stream_plan(const W4Params& p) {
    const int blocks = ceil_div(p.K, 128), eight = ceil_div(blocks, ceil_div(blocks, 8)), sixteen = ceil_div(blocks, ceil_div(blocks, 16));
    const int tiles = ceil_div(p.N, 16), sms = sm_count();
    if (stream_smem(p, eight, 1) > 232448) return {0, 0};
    if (4 * (stream_smem(p, eight, 1) + 1024) <= 233472) return {eight, 1};
    if (stream_smem(p, eight, 2) <= 232448 && 2 * ceil_div(tiles, 2 * sms) == ceil_div(tiles, sms)) return {eight, 2};
    return {stream_smem(p, sixteen, 1) <= 232448 ? sixteen : eight, 1};
}

template <bool WIDE, int TEAMS>
static int launch_stream(const W4Params& p, int warps, bool xaligned, cudaStream_t st) {
    const size_t smem = (size_t)stream_smem(p, warps, TEAMS);
    auto kernel = p.zero ? linear_w4_stream_kernel<WIDE, true, TEAMS> : linear_w4_stream_kernel<WIDE, false, TEAMS>;
    static bool attr_dev[KATZ_MAX_DEVICES][2] = {};
    bool& attr = attr_dev[current_device_index()][p.zero != nullptr];
    if (!attr) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
        if (e != cudaSuccess) return (int)e;
        attr = true;
    }
    // resident CTAs: 228 KB of shared memory an SM (1 KB of it per CTA), 64 registers a thread
    const int per_sm = std::max(1, std::min(1024 / (warps * TEAMS * 32), (int)(233472 / (smem + 1024))));
    launch_k(kernel, std::min(ceil_div(p.N, 16 * TEAMS), sm_count() * per_sm), warps * TEAMS * 32, smem, st, p, scale_rows(p, warps), xaligned);
    KATZ_LAUNCH_RET();
}

constexpr int W4_MAX_DIM = 1 << 30;      // indexes of tiles, and a little beyond, stay inside 32 bits

static int group_shift_of(int group) { return group == 32 ? 5 : group == 64 ? 6 : group == 128 ? 7 : -1; }

}  // namespace katz

using namespace katz;

extern "C" int katz_quantize_w4_f16(const void* w, long long ldw, void* q, void* scale, int N, int K, int group, void* stream) {
    KATZ_CHECK_ARG(w && q && scale, KATZ_EINVAL);
    const int shift = group_shift_of(group);
    KATZ_CHECK_ARG(shift > 0, KATZ_EINVAL);
    KATZ_CHECK_ARG(N > 0 && K > 0 && K % 32 == 0 && N <= W4_MAX_DIM && K <= W4_MAX_DIM && ldw >= K, KATZ_ESIZE);
    KATZ_CHECK_ARG(aligned16(w) && ldw % 8 == 0 && aligned16(q) && ((uintptr_t)scale & 1) == 0, KATZ_EALIGN);
    const PieceGrid g = piece_grid(N, K, group, ldw);
    KATZ_CHECK_ARG(g.ok, KATZ_ESIZE);
    auto kernel = group == 32 ? (g.flat ? quantize_w4_kernel<32, true> : quantize_w4_kernel<32, false>)
                  : group == 64 ? (g.flat ? quantize_w4_kernel<64, true> : quantize_w4_kernel<64, false>)
                                : (g.flat ? quantize_w4_kernel<128, true> : quantize_w4_kernel<128, false>);
    launch_k(kernel, g.ctas, 256, 0, (cudaStream_t)stream, (const __half*)w, ldw, (unsigned char*)q, (unsigned short*)scale, g.K,
             ceil_div(K, group), g.total, g.per_row);
    KATZ_LAUNCH_RET();
}

extern "C" int katz_dequantize_w4_f16(const void* q, const void* scale, const void* zero, void* w, long long ldw, int N, int K, int group,
                                      void* stream) {
    KATZ_CHECK_ARG(w && q && scale, KATZ_EINVAL);
    const int shift = group_shift_of(group);
    KATZ_CHECK_ARG(shift > 0, KATZ_EINVAL);
    KATZ_CHECK_ARG(N > 0 && K > 0 && K % 32 == 0 && N <= W4_MAX_DIM && K <= W4_MAX_DIM && ldw >= K, KATZ_ESIZE);
    KATZ_CHECK_ARG(aligned16(w) && ldw % 8 == 0 && aligned16(q) && ((uintptr_t)scale & 1) == 0, KATZ_EALIGN);
    const PieceGrid g = piece_grid(N, K, group, ldw);
    KATZ_CHECK_ARG(g.ok, KATZ_ESIZE);
    auto kernel = group == 32 ? (g.flat ? dequantize_w4_kernel<32, true> : dequantize_w4_kernel<32, false>)
                  : group == 64 ? (g.flat ? dequantize_w4_kernel<64, true> : dequantize_w4_kernel<64, false>)
                                : (g.flat ? dequantize_w4_kernel<128, true> : dequantize_w4_kernel<128, false>);
    launch_k(kernel, g.ctas, 256, 0, (cudaStream_t)stream, (const unsigned char*)q, (const unsigned short*)scale, (const unsigned char*)zero,
             (__half*)w, ldw, g.K, ceil_div(K, group), g.total, g.per_row);
    KATZ_LAUNCH_RET();
}

extern "C" int katz_linear_w4_f16(const katz_linear_w4_args* a, void* stream) {
    KATZ_CHECK_ARG(a && a->x && a->q && a->scale && a->out, KATZ_EINVAL);
    KATZ_CHECK_ARG(a->act == KATZ_ACT_NONE || a->act == KATZ_ACT_SILU, KATZ_EINVAL);
    const int shift = group_shift_of(a->group), M = a->M, N = a->N, K = a->K;
    KATZ_CHECK_ARG(shift > 0, KATZ_EINVAL);
    KATZ_CHECK_ARG(M > 0 && N > 0 && K > 0 && K % 32 == 0 && M <= W4_MAX_DIM && N <= W4_MAX_DIM && K <= W4_MAX_DIM, KATZ_ESIZE);
    KATZ_CHECK_ARG(M == 1 || (a->ldx >= K && a->ldo >= N && (!a->residual || a->ldr >= N)), KATZ_ESIZE);
    KATZ_CHECK_ARG(aligned16(a->q) && (((uintptr_t)a->scale | (uintptr_t)a->x | (uintptr_t)a->out | (uintptr_t)a->bias | (uintptr_t)a->residual) & 1) == 0,
                   KATZ_EALIGN);
    W4Params p{};
    p.x = (const __half*)a->x; p.q = (const unsigned char*)a->q; p.scale = (const unsigned short*)a->scale; p.zero = (const unsigned char*)a->zero;
    p.bias = (const __half*)a->bias; p.residual = (const __half*)a->residual; p.out = (__half*)a->out;
    p.ldx = a->ldx; p.ldo = a->ldo; p.ldr = a->ldr;
    p.M = M; p.N = N; p.K = K; p.J = ceil_div(K, a->group); p.group_shift = shift;
    p.act = a->act; p.out_scale = a->out_scale;
    const bool xaligned = aligned16(p.x) && (M == 1 || p.ldx % 8 == 0);
    cudaStream_t st = (cudaStream_t)stream;
    // Up to eight rows: direct while a warp's whole reduction is in flight at once or the weights are few, else streamed (weights
    // cold, direct / streamed, one row: 1280 x 1280 2.3 / 3.1 us, 40960 x 1280 13.9 / 14.1, 640 x 4096 3.6 / 3.8, 2560 x 2560
    // 6.2 / 5.0, 1280 x 5120 7.0 / 5.2, 8192 x 10240 21 / 17). More rows: direct while the rows, in sixteens, times the weights
    // are so few that the tcgen05 kernel's fixed 5 us are the longer (direct / tcgen05, rows x N x K: 77 x 640 x 640 3.2 / 7.4 us,
    // 300 x 320 x 320 3.2 / 6.7, 512 x 1280 x 320 8.3 / 7.0, 16 x 1280 x 1280 3.1 / 6.7, 64 x 1280 x 1280 5.2 / 7.0, 128 x 1280 x
    // 1280 7.1 / 7.6, 77 x 2560 x 1280 10.8 / 8.3, 16 x 10240 x 1280 7.7 / 8.8, 48 x 640 x 2560 4.6 / 7.0, 32 x 1280 x 2560 8.1 /
    // 7.3, 16 x 2560 x 5120 13.5 / 9.9). x that TMA cannot read takes the direct kernel at any size.
    const bool tc05 = xaligned && K >= W4_TC05_MIN_K;
    const long long weights = (long long)N * K;
    const bool streams = M <= 8 && K > 1280 && weights > 3000000;
    const StreamPlan plan = streams ? stream_plan(p) : StreamPlan{0, 0};
    if (plan.warps) {
        if (shift == 7) return plan.teams == 2 ? launch_stream<true, 2>(p, plan.warps, xaligned, st) : launch_stream<true, 1>(p, plan.warps, xaligned, st);
        return plan.teams == 2 ? launch_stream<false, 2>(p, plan.warps, xaligned, st) : launch_stream<false, 1>(p, plan.warps, xaligned, st);
    }
    const long long work = (long long)ceil_div(M, 16) * weights;
    if (tc05 && (M > 8 ? work > (K > 1280 ? 6000000 : K > 640 ? 14000000 : 10000000) : streams)) return linear_w4_tc05(p, st);
    return M <= 8 ? launch_direct<1>(p, xaligned, st) : launch_direct<2>(p, xaligned, st);
}
