// 4-bit weights with group scales (w4.cuh has the format): made from fp16 weights, read back, and multiplied with few rows.
#include <algorithm>

#include "tc05.cuh"      // packed fp32 arithmetic
#include "w4.cuh"
#include "katz_b200.h"

namespace katz {

using namespace w4;

// ---------------------------------------------------------------------------------------------------------------------
// fp16 -> codes and scales. Per group: scale = bf16(max |w| / 7), code = 8 + rint(w / scale) with ties to even. The quotient
// is the correctly rounded one (a product with the reciprocal and one residual step): w and scale have 11 and 8 significant
// bits, so a quotient that is not exactly half way between two codes is at least 2^-13 of its size away from there, and one
// that is comes out exact. |w / scale| <= 7 * (1 + 2^-8): no code leaves 1..15.
// A group that holds an infinity or a NaN gets a NaN scale: what is read back of it is NaN, never a plausible number.
//
// Bound by HBM (2.5 bytes per weight and the scales), which leaves about ten instructions a weight. A lane holds 8 weights; a
// group is 4, 8 or 16 neighbouring lanes; a warp works on W4_PIECES pieces of 256 weights so that enough loads are in flight.
// FLAT (contiguous rows of whole groups): the matrix is one run of groups and no lane is idle at a row's end.
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
// Bound by the stream of codes from HBM and, close behind, by the instructions that turn codes into operands; so scales, x and
// the loop's bookkeeping are kept out of those.
// A CTA owns 16 * RT weight rows and up to 8 * MT rows of x; its warps take turns over blocks of 128 k. Lane (g = lane / 4, t =
// lane % 4) holds the codes of weight rows g and g + 8 as four words of eight k; a word of each row makes the A operands of two
// m16n8k16 products. The sum over k may be taken in any order as long as both operands use the same one, so the codes are used
// as they lie in memory, and x is laid out to match once per CTA, in shared memory: the pairs (k, k + 4) that the unpacking
// gives, 16 bytes a lane and word, no two lanes in one bank. Which k a lane's words cover is chosen by the group size so that
// the four lanes of a row stay inside ONE group (a lane reads 16, 8 or 4 bytes at a time): a group's products are integers
// times x, exactly, and its scale multiplies the fp32 sum. CTAs are persistent. Each warp streams its codes through a ring in
// shared memory with asynchronous copies, across row tiles, every lane reading back what it copied itself: the bytes in
// flight that HBM needs (some 45 KB an SM) do not fit in registers (one block ahead in registers: 2.8 TB/s). Scales and zero
// points of a tile lie in shared memory, read row by row while the tile before is multiplied: gathered by the lanes that use
// them they took more tag lookups than the codes. The warps' sums meet in shared memory, added in warp order.
constexpr int W4_ROWS_THREADS = 512;
constexpr int W4_RING = 4;                    // blocks of a warp in flight or in use

// 16, 8 or 4 bytes of codes, global -> shared, zeros if !in. L2 fetches the 256 bytes around them, most of which the CTA's
// other warps are about to ask for: a row at a time a warp reads 64 bytes, and HBM gives such pieces at half its rate.
template <int BYTES>
__device__ __forceinline__ void copy_codes(uint32_t dst, const unsigned char* src, bool in) {
    const int n = in ? BYTES : 0;
    if (BYTES == 16) asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
    else asm volatile("cp.async.ca.shared.global.L2::256B [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(n), "n"(BYTES) : "memory");
}

// stride of a row of scales in shared memory: an odd number of 4-byte words, so that eight rows lie in different banks
static __host__ __device__ inline int scale_stride(int J) { return (J + 1) / 2 % 2 ? (J + 1) / 2 * 2 : (J + 1) / 2 * 2 + 2; }
// bytes of a row of x in shared memory: neighbouring rows 64 bytes apart modulo 128
static __host__ __device__ inline int x_row_bytes(int K) { return (K + 127) / 128 * 256 + 64; }

// where word i of lane t lies in a block of 128 k, and the reverse for a multiple of eight k
template <int GROUP>
struct Words {
    static constexpr int GROUPS = 128 / GROUP, PER_GROUP = 4 / GROUPS;      // groups a block, words a group
    static __device__ __forceinline__ int k(int i, int t) { return (i / PER_GROUP) * GROUP + t * (8 * PER_GROUP) + 8 * (i % PER_GROUP); }
    static __device__ __forceinline__ int slot(int k) {      // 4 i + t
        const int r = k % GROUP;
        return 4 * ((k / GROUP) * PER_GROUP + r / 8 % PER_GROUP) + r / (8 * PER_GROUP);
    }
};

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

template <int MT, int GROUP, bool ZERO>
__global__ void __launch_bounds__(W4_ROWS_THREADS) linear_w4_rows_kernel(const W4Params p, int rows_per_cta, bool xaligned) {
    typedef Words<GROUP> W;
    extern __shared__ __align__(16) unsigned char rows_smem[];
    constexpr int LD = 16 + 4;
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int m0 = blockIdx.y * rows_per_cta, rows = min(rows_per_cta, p.M - m0);
    const int sld = scale_stride(p.J), blocks = (p.K + 127) / 128, xld = x_row_bytes(p.K), tiles = (p.N + 15) / 16;
    unsigned char* xs = rows_smem;                                                        // [rows][xld]
    unsigned char* ring = xs + rows_per_cta * xld;                                        // [warp][W4_RING][2 rows][lane][16 bytes]
    float* red = reinterpret_cast<float*>(ring + warps * W4_RING * 1024);                 // [warp][8 * MT][LD]
    unsigned short* scales = reinterpret_cast<unsigned short*>(red + warps * 8 * MT * LD);      // [2][16][sld]
    unsigned char* zeros = reinterpret_cast<unsigned char*>(scales + 2 * 16 * sld);             // [2][16][sld]
    const uint32_t mine_at = smem_u32(ring) + warp * W4_RING * 1024 + lane * 16;
    // the next block to copy: of this warp's blocks of tile ctile the one at ck, whose codes of this lane lie at src[]
    int ctile = blockIdx.x, ck = warp;
    uint32_t cslot = 0;
    const unsigned char* src[2];
    auto at_tile = [&]() {
#pragma unroll
        for (int h = 0; h < 2; ++h)      // rows past the last are computed and not stored
            src[h] = p.q + (size_t)min(ctile * 16 + 8 * h + g, p.N - 1) * (p.K / 2) + warp * 64 + 4 * W::PER_GROUP * t;
    };
    at_tile();
    auto copy_next = [&]() {
        if (ctile < tiles) {
            // K is a multiple of 32: all of what a lane copies at a time exists, or none (only the last block lacks any)
            const int left = p.K - ck * 128;
#pragma unroll
            for (int j = 0; j < W::GROUPS; ++j) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t dst = mine_at + cslot + h * 512 + j * 4 * W::PER_GROUP;
                    if (left >= 128) copy_codes<4 * W::PER_GROUP>(dst, src[h] + j * (GROUP / 2), true);
                    else {
                        const bool in = W::k(j * W::PER_GROUP, t) < left;
                        copy_codes<4 * W::PER_GROUP>(dst, in ? src[h] + j * (GROUP / 2) : p.q, in);
                    }
                }
            }
            ck += warps;
            src[0] += warps * 64;
            src[1] += warps * 64;
            if (ck >= blocks) {
                ck = warp;
                ctile += gridDim.x;
                at_tile();
            }
        }
        cp_async_commit();
        cslot = (cslot + 1024) % (W4_RING * 1024);
    };
    auto read_scales = [&](int tile, int buf) {
        for (int r = warp; r < 16; r += warps) {
            const size_t at = (size_t)min(tile * 16 + r, p.N - 1) * p.J;
            for (int j = lane; j < p.J; j += 32) {
                scales[(buf * 16 + r) * sld + j] = __ldg(p.scale + at + j);
                if (ZERO) zeros[(buf * 16 + r) * sld + j] = __ldg(p.zero + at + j);
            }
        }
    };
    pdl_wait();
    pdl_launch_dependents();
#pragma unroll
    for (int i = 0; i < W4_RING - 1; ++i) copy_next();
    read_scales(blockIdx.x, 0);
    for (int v = threadIdx.x; v < blocks * 16; v += blockDim.x) {
        const int k = v * 8;
        for (int m = 0; m < rows; ++m)
            *reinterpret_cast<uint4*>(xs + m * xld + (k / 128 * 16 + W::slot(k % 128)) * 16) =
                k < p.K ? load_x_pairs(p.x + (m0 + m) * p.ldx + k, xaligned) : make_uint4(0, 0, 0, 0);
    }
    __syncthreads();
    // columns of x past the last row hold another row: what they give is not stored
    const uint32_t x_mine = smem_u32(xs) + 16 * t;
    uint32_t x_row[MT];
#pragma unroll
    for (int c = 0; c < MT; ++c) x_row[c] = x_mine + min(8 * c + g, rows - 1) * xld;
    uint32_t slot = 0;
    int buf = 0;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, buf ^= 1) {
        if (tile + (int)gridDim.x < tiles) read_scales(tile + gridDim.x, buf ^ 1);      // seen after this tile's barriers
        const unsigned short* s_row = scales + (buf * 16 + g) * sld;
        const unsigned char* z_row = zeros + (buf * 16 + g) * sld;
        float acc[MT][4] = {};
        for (int kb = warp; kb < blocks; kb += warps) {
            cp_async_wait<W4_RING - 2>();
            const uint4 v4[2] = {lds128(mine_at + slot), lds128(mine_at + slot + 512)};
            slot = (slot + 1024) % (W4_RING * 1024);
            copy_next();      // into the slot that was read in the round before
            const uint32_t v[2][4] = {{v4[0].x, v4[0].y, v4[0].z, v4[0].w}, {v4[1].x, v4[1].y, v4[1].z, v4[1].w}};
#pragma unroll
            for (int j = 0; j < W::GROUPS; ++j) {
                float part[MT][2][4];      // two chains of products
                const int jg = min(kb * W::GROUPS + j, p.J - 1);      // past the last k x is zero
                __half2 low[2], high[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    low[h] = as_half2(0xe408e408u);       // -(1024 + 8)
                    high[h] = as_half2(0xd480d480u);      // -(64 + 8)
                    if (ZERO) {
                        const uint32_t z = z_row[8 * h * sld + jg];
                        low[h] = as_half2(0xe400e400u + z * 0x00010001u);
                        high[h] = as_half2(0xd400d400u + z * 0x00100010u);
                    }
                }
#pragma unroll
                for (int i = j * W::PER_GROUP; i < (j + 1) * W::PER_GROUP; ++i) {
                    __half2 lo[4], hi[4];
                    unpack8(v[0][i], low[0], high[0], lo);
                    unpack8(v[1][i], low[1], high[1], hi);
                    const uint32_t a0[4] = {as_u32(lo[0]), as_u32(hi[0]), as_u32(lo[1]), as_u32(hi[1])};
                    const uint32_t a1[4] = {as_u32(lo[2]), as_u32(hi[2]), as_u32(lo[3]), as_u32(hi[3])};
#pragma unroll
                    for (int c = 0; c < MT; ++c) {
                        const uint4 b = lds128(x_row[c] + (kb * 4 + i) * 64);
                        const uint32_t b0[2] = {b.x, b.y}, b1[2] = {b.z, b.w};
                        if (i % W::PER_GROUP == 0) {
                            mma_f16_16816_first(part[c][0], a0, b0);
                            mma_f16_16816_first(part[c][1], a1, b1);
                        } else {
                            mma_f16_16816(part[c][0], a0, b0);
                            mma_f16_16816(part[c][1], a1, b1);
                        }
                    }
                }
                const float sl = bf16_bits_to_float(s_row[jg]), sh = bf16_bits_to_float(s_row[8 * sld + jg]);
#pragma unroll
                for (int c = 0; c < MT; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[c][e] = fmaf(e < 2 ? sl : sh, part[c][0][e] + part[c][1][e], acc[c][e]);
            }
        }
#pragma unroll
        for (int c = 0; c < MT; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) red[(warp * 8 * MT + 8 * c + 2 * t + (e & 1)) * LD + g + 8 * (e >> 1)] = acc[c][e];
        __syncthreads();
        for (int i = threadIdx.x; i < rows * 16; i += blockDim.x) {
            const int ml = i / 16, nl = i % 16, n = tile * 16 + nl;
            const long long m = m0 + ml;
            if (n >= p.N) continue;
            float v = 0.f;
            for (int w = 0; w < warps; ++w) v += red[(w * 8 * MT + ml) * LD + nl];
            if (p.bias) v += __half2float(p.bias[n]);
            if (p.act == KATZ_ACT_SILU) v = silu_f(v);
            if (p.residual) v += __half2float(p.residual[m * p.ldr + n]);
            p.out[m * p.ldo + n] = __float2half_rn(v * p.out_scale);
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

struct RowsLaunch {
    int rows, warps;      // of x a CTA
    size_t smem;
};
// false: K is too long for even one row of x and its scales in shared memory
static bool rows_launch(const W4Params& p, RowsLaunch& l) {
    const int mt = p.M <= 8 ? 1 : 2, blocks = ceil_div(p.K, 128);
    for (int most = 8; most <= W4_ROWS_THREADS / 32; most += 8) {
        // as many warps as share the blocks of k evenly
        l.warps = ceil_div(blocks, ceil_div(blocks, most));
        const long long fixed = (long long)l.warps * (W4_RING * 1024 + 8 * mt * 20 * 4) + 2ll * 16 * scale_stride(p.J) * (p.zero ? 3 : 2);
        const long long fit = (232448 - fixed) / x_row_bytes(p.K);
        if (fixed >= 232448 || fit < 1) return false;
        l.rows = (int)std::min<long long>(std::min(p.M, 8 * mt), fit);
        l.smem = (size_t)(fixed + (long long)l.rows * x_row_bytes(p.K));
        // Eight warps a CTA where four such CTAs fit an SM: what a tile costs outside its blocks (barriers, sums, scales) is
        // spread over twice as many of them. With more x in shared memory, or too few tiles to go round, sixteen.
        if (4 * (l.smem + 1024) <= 233472 && ceil_div(p.N, 16) >= 2 * sm_count()) break;
    }
    return true;
}

template <int MT, int GROUP>
static int launch_rows(const W4Params& p, const RowsLaunch& l, bool xaligned, cudaStream_t st) {
    const int row_blocks = ceil_div(p.M, l.rows);
    KATZ_CHECK_ARG(row_blocks <= 65535, KATZ_ESIZE);
    auto kernel = p.zero ? linear_w4_rows_kernel<MT, GROUP, true> : linear_w4_rows_kernel<MT, GROUP, false>;
    static bool attr_dev[KATZ_MAX_DEVICES][2] = {};
    bool& attr = attr_dev[current_device_index()][p.zero != nullptr];
    if (!attr) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
        if (e != cudaSuccess) return (int)e;
        attr = true;
    }
    // resident CTAs: 228 KB of shared memory an SM (1 KB of it per CTA), 64 registers a thread
    const int per_sm = std::max(1, std::min(1024 / (l.warps * 32), (int)(233472 / (l.smem + 1024))));
    const int slots = std::max(1, sm_count() * per_sm / row_blocks);
    launch_k(kernel, dim3(std::min(ceil_div(p.N, 16), slots), row_blocks), l.warps * 32, l.smem, st, p, l.rows, xaligned);
    KATZ_LAUNCH_RET();
}

template <int MT>
static int launch_rows(const W4Params& p, const RowsLaunch& l, bool xaligned, cudaStream_t st) {
    if (p.group_shift == 5) return launch_rows<MT, 32>(p, l, xaligned, st);
    if (p.group_shift == 6) return launch_rows<MT, 64>(p, l, xaligned, st);
    return launch_rows<MT, 128>(p, l, xaligned, st);
}

static int group_shift_of(int group) { return group == 32 ? 5 : group == 64 ? 6 : group == 128 ? 7 : -1; }

}  // namespace katz

using namespace katz;

extern "C" int katz_quantize_w4_f16(const void* w, long long ldw, void* q, void* scale, int N, int K, int group, void* stream) {
    KATZ_CHECK_ARG(w && q && scale, KATZ_EINVAL);
    const int shift = group_shift_of(group);
    KATZ_CHECK_ARG(shift > 0, KATZ_EINVAL);
    KATZ_CHECK_ARG(N > 0 && K > 0 && K % 32 == 0 && ldw >= K, KATZ_ESIZE);
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
    KATZ_CHECK_ARG(N > 0 && K > 0 && K % 32 == 0 && ldw >= K, KATZ_ESIZE);
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

extern "C" int katz_linear_w4_f16(const void* x, long long ldx, const void* q, const void* scale, const void* zero, int group, void* out,
                                  long long ldo, int M, int N, int K, const void* bias, const void* residual, long long ldr, int act,
                                  float out_scale, void* stream) {
    KATZ_CHECK_ARG(x && q && scale && out, KATZ_EINVAL);
    KATZ_CHECK_ARG(act == KATZ_ACT_NONE || act == KATZ_ACT_SILU, KATZ_EINVAL);
    const int shift = group_shift_of(group);
    KATZ_CHECK_ARG(shift > 0, KATZ_EINVAL);
    KATZ_CHECK_ARG(M > 0 && N > 0 && K > 0 && K % 32 == 0, KATZ_ESIZE);
    KATZ_CHECK_ARG((M == 1 || ldx >= K) && (M == 1 || ldo >= N) && (M == 1 || !residual || ldr >= N), KATZ_ESIZE);
    KATZ_CHECK_ARG(aligned16(q) && ((uintptr_t)scale & 1) == 0 && (((uintptr_t)x | (uintptr_t)out | (uintptr_t)bias | (uintptr_t)residual) & 1) == 0,
                   KATZ_EALIGN);
    W4Params p{};
    p.x = (const __half*)x; p.q = (const unsigned char*)q; p.scale = (const unsigned short*)scale; p.zero = (const unsigned char*)zero;
    p.bias = (const __half*)bias; p.residual = (const __half*)residual; p.out = (__half*)out;
    p.ldx = ldx; p.ldo = ldo; p.ldr = ldr;
    p.M = M; p.N = N; p.K = K; p.J = ceil_div(K, group); p.group_shift = shift;
    p.act = act; p.out_scale = out_scale;
    const bool xaligned = aligned16(x) && (M == 1 || ldx % 8 == 0);
    cudaStream_t st = (cudaStream_t)stream;
    // Few rows go to the kernel of this file while all of x fits shared memory at once: up to 8 rows always (8 x 8192 x 8192:
    // 20.2 us here, 20.0 us on the tcgen05 path; 8 x 5120 x 1280: 5.8 and 7.9 us; but 8 x 1280 x 10240, where x takes two
    // turns: 14.0 and 10.8 us), up to 16 for small weights (16 x 1280 x 1280: 4.5 and 7.0 us, 16 x 5120 x 1280: 7.3 and 7.9 us, 16 x
    // 10240 x 1280: 9.8 and 8.6 us, 16 x 8192 x 8192: 40.7 and 20.0 us). Rows of x that TMA cannot read stay here whatever M.
    RowsLaunch l;
    const bool rows = rows_launch(p, l), tc05 = xaligned && K >= W4_TC05_MIN_K;
    const bool few = rows && l.rows >= M && (M <= 8 || (M <= 16 && (long long)N * K <= 8000000));
    if (tc05 && !few) return linear_w4_tc05(p, st);
    KATZ_CHECK_ARG(rows, KATZ_ESIZE);
    return M <= 8 ? launch_rows<1>(p, l, xaligned, st) : launch_rows<2>(p, l, xaligned, st);
}
