// 4-bit weights with group scales (w4.cuh has the format): made from fp16 weights, read back, and multiplied with few rows.
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
// Bound by HBM (2.5 bytes per weight and the scales). A lane holds 8 weights; a group is 4, 8 or 16 neighbouring lanes; a
// warp works on W4_PIECES pieces of 256 weights at a time so that enough loads are in flight.
constexpr int W4_PIECES = 4;

__device__ __forceinline__ __half2 hmax2_abs_nan(__half2 a, __half2 b) { return __hmax2_nan(__habs2(a), __habs2(b)); }

template <int GROUP>
__global__ void __launch_bounds__(256) quantize_w4_kernel(const __half* __restrict__ w, long long ldw, unsigned char* __restrict__ q,
                                                          unsigned short* __restrict__ scale, int N, int K, int J,
                                                          int pieces_per_row) {
    pdl_wait();      // writes weights: the next kernel is not released early
    constexpr int LANES = GROUP / 8;
    const int lane = threadIdx.x & 31;
    const long long total = (long long)N * pieces_per_row;
    const long long first = ((long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * W4_PIECES;
    long long row = first / pieces_per_row;
    int piece = (int)(first - row * pieces_per_row);
    uint4 v[W4_PIECES];
    long long rows[W4_PIECES];
    int ks[W4_PIECES];
#pragma unroll
    for (int i = 0; i < W4_PIECES; ++i) {
        rows[i] = first + i < total ? row : -1;
        ks[i] = piece * 256 + lane * 8;
        v[i] = make_uint4(0, 0, 0, 0);
        if (rows[i] >= 0 && ks[i] < K) v[i] = __ldg(reinterpret_cast<const uint4*>(w + row * ldw + ks[i]));
        if (++piece == pieces_per_row) {
            piece = 0;
            ++row;
        }
    }
#pragma unroll
    for (int i = 0; i < W4_PIECES; ++i) {
        if (rows[i] < 0) return;      // uniform over the warp
        const uint32_t u[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
        __half2 m2 = hmax2_abs_nan(hmax2_abs_nan(as_half2(u[0]), as_half2(u[1])), hmax2_abs_nan(as_half2(u[2]), as_half2(u[3])));
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) m2 = hmax2_abs_nan(m2, as_half2(__shfl_xor_sync(0xffffffffu, as_u32(m2), o)));
        const float top = __half2float(__hmax_nan(__low2half(m2), __high2half(m2)));
        __nv_bfloat16 sb = __float2bfloat16_rn(__fdiv_rn(top, 7.0f));
        if (!(top <= 65504.0f)) sb = __float2bfloat16_rn(__uint_as_float(0x7fc00000u));
        const float s = __bfloat162float(sb);
        const float inv = s > 0.f ? __frcp_rn(s) : 0.f;
        uint32_t codes = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 f = unpack_half2(u[e]);
            float t0 = f.x * inv, t1 = f.y * inv;
            t0 = fmaf(fmaf(-t0, s, f.x), inv, t0);
            t1 = fmaf(fmaf(-t1, s, f.y), inv, t1);
            // adding 1.5 * 2^23 rounds to an integer (ties to even) and leaves it in the low bits; 8 is the code of zero
            const uint32_t c0 = __float_as_uint(t0 + 12582912.0f) + 8u, c1 = __float_as_uint(t1 + 12582912.0f) + 8u;
            codes |= ((c0 & 15u) | ((c1 & 15u) << 4)) << (8 * e);
        }
        if (ks[i] < K) {
            *reinterpret_cast<uint32_t*>(q + rows[i] * (K / 2) + ks[i] / 2) = codes;
            if ((lane & (LANES - 1)) == 0) scale[rows[i] * J + ks[i] / GROUP] = __bfloat16_as_ushort(sb);
        }
    }
}

// codes, scales -> fp16(scale * (code - zero)), one rounding. Bound by HBM (2.5 bytes per weight); the same shape as above.
__global__ void __launch_bounds__(256) dequantize_w4_kernel(const unsigned char* __restrict__ q, const unsigned short* __restrict__ scale,
                                                            const unsigned char* __restrict__ zero, __half* __restrict__ w,
                                                            long long ldw, int N, int K, int J, int group_shift, int pieces_per_row) {
    pdl_wait();      // writes weights: the next kernel is not released early
    const int lane = threadIdx.x & 31;
    const long long total = (long long)N * pieces_per_row;
    const long long first = ((long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * W4_PIECES;
    long long row = first / pieces_per_row;
    int piece = (int)(first - row * pieces_per_row);
    uint32_t v[W4_PIECES];
    unsigned short sb[W4_PIECES];
    unsigned char zb[W4_PIECES];
    __half* dst[W4_PIECES];
#pragma unroll
    for (int i = 0; i < W4_PIECES; ++i) {
        const int k = piece * 256 + lane * 8;
        const bool in = first + i < total && k < K;
        dst[i] = in ? w + row * ldw + k : nullptr;
        v[i] = in ? __ldg(reinterpret_cast<const uint32_t*>(q + row * (K / 2) + k / 2)) : 0u;
        sb[i] = in ? __ldg(scale + row * J + (k >> group_shift)) : (unsigned short)0;
        zb[i] = in && zero ? __ldg(zero + row * J + (k >> group_shift)) : (unsigned char)8;
        if (++piece == pieces_per_row) {
            piece = 0;
            ++row;
        }
    }
#pragma unroll
    for (int i = 0; i < W4_PIECES; ++i) {
        if (!dst[i]) continue;
        __half2 d[4];
        unpack8(v[i], __float2half2_rn((float)(-1024 - (int)zb[i])), __float2half2_rn((float)(-64 - (int)zb[i])), d);
        const float s = bf16_bits_to_float(sb[i]);
        float2 f[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f[e] = __half22float2(d[e]);
            f[e].x *= s;
            f[e].y *= s;
        }
        *reinterpret_cast<uint4*>(dst[i]) = make_uint4(pack_half2(f[0].x, f[1].x), pack_half2(f[2].x, f[3].x), pack_half2(f[0].y, f[1].y),
                                                       pack_half2(f[2].y, f[3].y));
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Few rows: out[M, N] = (act(x W^T + bias) + residual) * out_scale with W in 4 bits.
//
// A CTA owns 16 * RT weight rows and 8 * MT rows of x; its warps take turns over blocks of 128 k. In a block a lane (g =
// lane / 4, t = lane % 4) reads 16 bytes of weight row g and of row g + 8 (the 32 k from 32 t on), which are its operand
// fragments of eight m16n8k16 products: the sum over k may be taken in any order as long as both operands use the same one,
// so nothing is rearranged in memory, a lane's 32 weights lie in one group, and the pairs (k, k + 4) that the unpacking
// gives are matched by pairing x with a byte permute. The warps' sums meet in shared memory, added in warp order.
constexpr int W4_ROWS_WARPS = 8;

template <int MT, int RT, bool XALIGNED>
__global__ void __launch_bounds__(W4_ROWS_WARPS * 32) linear_w4_rows_kernel(const W4Params p) {
    __shared__ float red[W4_ROWS_WARPS][8 * MT][16 * RT + 4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * 16 * RT, m0 = blockIdx.y * 8 * MT;
    float acc[RT][MT][4] = {};
    pdl_wait();
    pdl_launch_dependents();
    const int blocks = (p.K + 127) / 128;
    for (int kb = warp; kb < blocks; kb += W4_ROWS_WARPS) {
        const int k = kb * 128 + 32 * t;
        const bool k_in = k < p.K;      // K is a multiple of 32: a lane's 32 k exist together or not at all
        uint4 a[RT][2];
        Group grp[RT][2];
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int n = min(n0 + 16 * r + 8 * s + g, p.N - 1);      // rows past the last are computed and not stored
                a[r][s] = make_uint4(0, 0, 0, 0);
                unsigned short sb = 0;
                int z = 8;
                if (k_in) {
                    a[r][s] = __ldg(reinterpret_cast<const uint4*>(p.q + (size_t)n * (p.K / 2) + k / 2));
                    const size_t j = (size_t)n * p.J + (k >> p.group_shift);
                    sb = __ldg(p.scale + j);
                    if (p.zero) z = __ldg(p.zero + j);
                }
                grp[r][s] = make_group(sb, z);
            }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            uint32_t b[MT][4];
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int m = m0 + 8 * i + g;
                uint4 xv = make_uint4(0, 0, 0, 0);
                if (k_in && m < p.M) {
                    const __half* src = p.x + m * p.ldx + k + 8 * c;
                    if (XALIGNED) {
                        xv = *reinterpret_cast<const uint4*>(src);
                    } else {
                        const unsigned short* e = reinterpret_cast<const unsigned short*>(src);
                        xv = make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16,
                                        e[6] | (uint32_t)e[7] << 16);
                    }
                }
                b[i][0] = __byte_perm(xv.x, xv.z, 0x5410);
                b[i][1] = __byte_perm(xv.x, xv.z, 0x7632);
                b[i][2] = __byte_perm(xv.y, xv.w, 0x5410);
                b[i][3] = __byte_perm(xv.y, xv.w, 0x7632);
            }
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                uint32_t lo[4], hi[4];
                weights8(c == 0 ? a[r][0].x : c == 1 ? a[r][0].y : c == 2 ? a[r][0].z : a[r][0].w, grp[r][0], lo);
                weights8(c == 0 ? a[r][1].x : c == 1 ? a[r][1].y : c == 2 ? a[r][1].z : a[r][1].w, grp[r][1], hi);
                const uint32_t a0[4] = {lo[0], hi[0], lo[1], hi[1]}, a1[4] = {lo[2], hi[2], lo[3], hi[3]};
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    mma_f16_16816(acc[r][i], a0, b[i]);
                    mma_f16_16816(acc[r][i], a1, b[i] + 2);
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) red[warp][8 * i + 2 * t + (e & 1)][16 * r + g + 8 * (e >> 1)] = acc[r][i][e];
    __syncthreads();
    for (int i = threadIdx.x; i < 8 * MT * 16 * RT; i += W4_ROWS_WARPS * 32) {
        const int ml = i / (16 * RT), nl = i % (16 * RT), m = m0 + ml, n = n0 + nl;
        if (m >= p.M || n >= p.N) continue;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < W4_ROWS_WARPS; ++w) v += red[w][ml][nl];
        p.out[m * p.ldo + n] = __float2half_rn(w4_epilogue(p, v, m, n));
    }
}

template <int MT, int RT>
static void launch_rows(const W4Params& p, bool xaligned, cudaStream_t st) {
    const dim3 grid(ceil_div(p.N, 16 * RT), ceil_div(p.M, 8 * MT));
    if (xaligned) launch_k(linear_w4_rows_kernel<MT, RT, true>, grid, W4_ROWS_WARPS * 32, 0, st, p);
    else launch_k(linear_w4_rows_kernel<MT, RT, false>, grid, W4_ROWS_WARPS * 32, 0, st, p);
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
    const int pieces = ceil_div(K, 256);
    const long long ctas = ceil_div_ll((long long)N * pieces, 8 * W4_PIECES);
    KATZ_CHECK_ARG(ctas < (1ll << 31), KATZ_ESIZE);
    const int J = ceil_div(K, group);
    auto kernel = group == 32 ? quantize_w4_kernel<32> : group == 64 ? quantize_w4_kernel<64> : quantize_w4_kernel<128>;
    launch_k(kernel, (unsigned)ctas, 256, 0, (cudaStream_t)stream, (const __half*)w, ldw, (unsigned char*)q, (unsigned short*)scale, N, K,
             J, pieces);
    KATZ_LAUNCH_RET();
}

extern "C" int katz_dequantize_w4_f16(const void* q, const void* scale, const void* zero, void* w, long long ldw, int N, int K, int group,
                                      void* stream) {
    KATZ_CHECK_ARG(w && q && scale, KATZ_EINVAL);
    const int shift = group_shift_of(group);
    KATZ_CHECK_ARG(shift > 0, KATZ_EINVAL);
    KATZ_CHECK_ARG(N > 0 && K > 0 && K % 32 == 0 && ldw >= K, KATZ_ESIZE);
    KATZ_CHECK_ARG(aligned16(w) && ldw % 8 == 0 && aligned16(q) && ((uintptr_t)scale & 1) == 0, KATZ_EALIGN);
    const int pieces = ceil_div(K, 256);
    const long long ctas = ceil_div_ll((long long)N * pieces, 8 * W4_PIECES);
    KATZ_CHECK_ARG(ctas < (1ll << 31), KATZ_ESIZE);
    launch_k(dequantize_w4_kernel, (unsigned)ctas, 256, 0, (cudaStream_t)stream, (const unsigned char*)q, (const unsigned short*)scale,
             (const unsigned char*)zero, (__half*)w, ldw, N, K, ceil_div(K, group), shift, pieces);
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
    KATZ_CHECK_ARG(ceil_div(M, 32) <= 65535, KATZ_ESIZE);
    const bool xaligned = aligned16(x) && (M == 1 || ldx % 8 == 0);
    cudaStream_t st = (cudaStream_t)stream;
    if (M > 16 && xaligned && K >= W4_TC05_MIN_K) return linear_w4_tc05(p, st);
    if (M <= 8) launch_rows<1, 1>(p, xaligned, st);
    else if (M <= 16) launch_rows<2, 1>(p, xaligned, st);
    else launch_rows<4, 2>(p, xaligned, st);
    KATZ_LAUNCH_RET();
}
