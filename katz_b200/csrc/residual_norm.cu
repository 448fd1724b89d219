// The norms after and before a block, with the block's gate and the residual scale between them, in one pass:
//   u = post(y)                    (LayerNorm, RMSNorm or none; y: the block's output)
//   h = residual_scale * x + gate * u
//   z = pre(h) * (1 + scale) + shift   (LayerNorm, RMSNorm or none: the next block's input)
// LayerNorm(v) = (v - mean) / sqrt(var + eps) * weight + bias, RMSNorm(v) = v / sqrt(mean of v^2 + eps) * weight + bias; weight and
// bias are optional, gate, scale and shift may be per channel, per sample or per token (strides of zero).
//
// Bound by HBM: x and y are read once, h and z written once, 8 bytes per element in fp16. A row stays in registers from the
// load to the store; statistics are fp32, of the values before any rounding (z is computed from the unrounded h), and the
// variance is the mean of squared differences from the mean, so a row whose mean is large loses nothing. Rows of up to 1280
// channels belong to one warp (sums by shuffles, no barrier), longer ones to 4 or 16 warps.
#include "common.cuh"

namespace katz {

struct ResidualNormParams {
    const void* x;
    const __half* y;
    const __half* gate;
    const __half* scale;
    const __half* shift;
    const __half* post_w;
    const __half* post_b;
    const __half* pre_w;
    const __half* pre_b;
    void* h;
    __half* z;
    long long x_sb, x_ss, y_sb, y_ss, h_sb, h_ss, z_sb, z_ss, gate_sb, gate_ss, scale_sb, scale_ss, shift_sb, shift_ss;
    int S, C;
    long long rows;
    int post_kind, pre_kind;
    float post_eps, pre_eps, residual_scale;
};

template <bool F32>
struct Stream;
template <>
struct Stream<false> { typedef __half T; };
template <>
struct Stream<true> { typedef float T; };

// T threads share a row; sums over all of them, the same value in every thread. `slot` alternates between two shared arrays.
template <int T>
__device__ __forceinline__ float row_sum(float v, float* red, int& slot) {
    v = warp_sum(v);
    if constexpr (T > 32) {
        float* r = red + slot * (T / 32);
        slot ^= 1;
        if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < T / 32; ++i) v += r[i];
    }
    return v;
}

// channel of element e of vector i
template <int T, bool VEC>
__device__ __forceinline__ int channel(int i, int e, int tid) {
    return VEC ? (i * T + tid) * 8 + e : (i * 8 + e) * T + tid;
}

template <int T, int NV, bool VEC>
__device__ __forceinline__ void load_row(const __half* src, int C, int tid, float (&v)[NV][8]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (VEC) {
            const int c = channel<T, VEC>(i, 0, tid);
            uint4 w = make_uint4(0, 0, 0, 0);
            if (c < C) w = *reinterpret_cast<const uint4*>(src + c);
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 f = unpack_half2(u[e]);
                v[i][2 * e] = f.x;
                v[i][2 * e + 1] = f.y;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int c = channel<T, VEC>(i, e, tid);
                v[i][e] = c < C ? __half2float(src[c]) : 0.f;
            }
        }
    }
}
template <int T, int NV, bool VEC>
__device__ __forceinline__ void load_row(const float* src, int C, int tid, float (&v)[NV][8]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (VEC) {
            const int c = channel<T, VEC>(i, 0, tid);
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
            if (c < C) {
                a = *reinterpret_cast<const float4*>(src + c);
                b = *reinterpret_cast<const float4*>(src + c + 4);
            }
            const float f[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = f[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int c = channel<T, VEC>(i, e, tid);
                v[i][e] = c < C ? src[c] : 0.f;
            }
        }
    }
}
template <int T, int NV, bool VEC>
__device__ __forceinline__ void store_row(__half* dst, int C, int tid, const float (&v)[NV][8]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (VEC) {
            const int c = channel<T, VEC>(i, 0, tid);
            if (c < C)
                *reinterpret_cast<uint4*>(dst + c) = make_uint4(pack_half2(v[i][0], v[i][1]), pack_half2(v[i][2], v[i][3]),
                                                                pack_half2(v[i][4], v[i][5]), pack_half2(v[i][6], v[i][7]));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int c = channel<T, VEC>(i, e, tid);
                if (c < C) dst[c] = __float2half_rn(v[i][e]);
            }
        }
    }
}
template <int T, int NV, bool VEC>
__device__ __forceinline__ void store_row(float* dst, int C, int tid, const float (&v)[NV][8]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (VEC) {
            const int c = channel<T, VEC>(i, 0, tid);
            if (c < C) {
                *reinterpret_cast<float4*>(dst + c) = make_float4(v[i][0], v[i][1], v[i][2], v[i][3]);
                *reinterpret_cast<float4*>(dst + c + 4) = make_float4(v[i][4], v[i][5], v[i][6], v[i][7]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int c = channel<T, VEC>(i, e, tid);
                if (c < C) dst[c] = v[i][e];
            }
        }
    }
}

// v <- normalised v (weight and bias applied)
template <int T, int NV, bool VEC>
__device__ __forceinline__ void normalise(float (&v)[NV][8], int kind, const __half* weight, const __half* bias, float eps, int C, int tid,
                                          float* red, int& slot) {
    const float inv_c = 1.0f / (float)C;
    float mean = 0.f;
    if (kind == KATZ_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) s += v[i][e];      // channels past the last hold zeros
        mean = row_sum<T>(s, red, slot) * inv_c;
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float d = v[i][e] - mean;
            if (channel<T, VEC>(i, e, tid) < C) q = fmaf(d, d, q);
        }
    const float rstd = rsqrtf(row_sum<T>(q, red, slot) * inv_c + eps);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = (v[i][e] - mean) * rstd;
    if (weight) {
        float g[NV][8];
        load_row<T, NV, VEC>(weight, C, tid, g);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] *= g[i][e];
    }
    if (bias) {
        float b[NV][8];
        load_row<T, NV, VEC>(bias, C, tid, b);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] += b[i][e];
    }
}

// one row per T threads; a CTA of max(T, 128) threads
template <int T, int NV, bool VEC, bool F32>
__global__ void __launch_bounds__(T > 128 ? T : 128) residual_norm_kernel(const ResidualNormParams p) {
    typedef typename Stream<F32>::T XT;
    __shared__ float red[2 * (T > 32 ? T / 32 : 1)];
    constexpr int ROWS = T >= 128 ? 1 : 128 / T;
    pdl_wait();
    pdl_launch_dependents();
    const int tid = threadIdx.x % T;
    const long long row = (long long)blockIdx.x * ROWS + threadIdx.x / T;
    if (row >= p.rows) return;      // uniform over the threads of a row
    const long long b = row / p.S, s = row - b * p.S;
    int slot = 0;
    float h[NV][8];
    load_row<T, NV, VEC>(static_cast<const XT*>(p.x) + b * p.x_sb + s * p.x_ss, p.C, tid, h);
    if (p.y) {
        float u[NV][8];
        load_row<T, NV, VEC>(p.y + b * p.y_sb + s * p.y_ss, p.C, tid, u);
        if (p.post_kind != KATZ_NORM_NONE) normalise<T, NV, VEC>(u, p.post_kind, p.post_w, p.post_b, p.post_eps, p.C, tid, red, slot);
        if (p.gate) {
            float g[NV][8];
            load_row<T, NV, VEC>(p.gate + b * p.gate_sb + s * p.gate_ss, p.C, tid, g);
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) u[i][e] *= g[i][e];
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) h[i][e] = fmaf(p.residual_scale, h[i][e], u[i][e]);
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) h[i][e] *= p.residual_scale;
    }
    if (p.h) store_row<T, NV, VEC>(static_cast<XT*>(p.h) + b * p.h_sb + s * p.h_ss, p.C, tid, h);
    if (p.pre_kind == KATZ_NORM_NONE) return;
    normalise<T, NV, VEC>(h, p.pre_kind, p.pre_w, p.pre_b, p.pre_eps, p.C, tid, red, slot);
    if (p.scale) {
        float g[NV][8];
        load_row<T, NV, VEC>(p.scale + b * p.scale_sb + s * p.scale_ss, p.C, tid, g);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) h[i][e] = fmaf(h[i][e], g[i][e], h[i][e]);
    }
    if (p.shift) {
        float g[NV][8];
        load_row<T, NV, VEC>(p.shift + b * p.shift_sb + s * p.shift_ss, p.C, tid, g);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) h[i][e] += g[i][e];
    }
    store_row<T, NV, VEC>(p.z + b * p.z_sb + s * p.z_ss, p.C, tid, h);
}

template <int T, int NV, bool VEC>
static void launch_residual_norm(const ResidualNormParams& p, bool f32, cudaStream_t st) {
    constexpr int ROWS = T >= 128 ? 1 : 128 / T;
    const unsigned grid = (unsigned)ceil_div_ll(p.rows, ROWS);
    if (f32) launch_k(residual_norm_kernel<T, NV, VEC, true>, grid, T > 128 ? T : 128, 0, st, p);
    else launch_k(residual_norm_kernel<T, NV, VEC, false>, grid, T > 128 ? T : 128, 0, st, p);
}

template <bool VEC>
static void dispatch_residual_norm(const ResidualNormParams& p, bool f32, cudaStream_t st) {
    if (p.C <= 32 * 8) launch_residual_norm<32, 1, VEC>(p, f32, st);
    else if (p.C <= 32 * 16) launch_residual_norm<32, 2, VEC>(p, f32, st);
    else if (p.C <= 32 * 24) launch_residual_norm<32, 3, VEC>(p, f32, st);
    else if (p.C <= 32 * 40) launch_residual_norm<32, 5, VEC>(p, f32, st);
    else if (p.C <= 128 * 16) launch_residual_norm<128, 2, VEC>(p, f32, st);
    else if (p.C <= 128 * 32) launch_residual_norm<128, 4, VEC>(p, f32, st);
    else if (p.C <= 512 * 16) launch_residual_norm<512, 2, VEC>(p, f32, st);
    else launch_residual_norm<512, 4, VEC>(p, f32, st);
}

}  // namespace katz

using namespace katz;

extern "C" int katz_residual_norm_f16(const katz_residual_norm_args* a, void* stream) {
    KATZ_CHECK_ARG(a && a->x, KATZ_EINVAL);
    KATZ_CHECK_ARG(a->x_dtype == KATZ_DTYPE_F16 || a->x_dtype == KATZ_DTYPE_F32, KATZ_EINVAL);
    KATZ_CHECK_ARG(a->post_kind >= KATZ_NORM_NONE && a->post_kind <= KATZ_NORM_RMS, KATZ_EINVAL);
    KATZ_CHECK_ARG(a->pre_kind >= KATZ_NORM_NONE && a->pre_kind <= KATZ_NORM_RMS, KATZ_EINVAL);
    KATZ_CHECK_ARG(a->y || (a->post_kind == KATZ_NORM_NONE && !a->gate), KATZ_EINVAL);
    KATZ_CHECK_ARG((a->pre_kind != KATZ_NORM_NONE) == (a->z != nullptr), KATZ_EINVAL);
    KATZ_CHECK_ARG(a->pre_kind != KATZ_NORM_NONE || (!a->scale && !a->shift), KATZ_EINVAL);
    KATZ_CHECK_ARG(a->h || a->z, KATZ_EINVAL);
    KATZ_CHECK_ARG(a->B > 0 && a->S > 0 && a->C > 0 && a->C <= KATZ_RESIDUAL_NORM_MAX_C, KATZ_ESIZE);
    const long long rows = (long long)a->B * a->S;
    KATZ_CHECK_ARG(rows < (1ll << 31), KATZ_ESIZE);
    const bool f32 = a->x_dtype == KATZ_DTYPE_F32;
    const uintptr_t half_ptrs = (uintptr_t)a->y | (uintptr_t)a->gate | (uintptr_t)a->scale | (uintptr_t)a->shift | (uintptr_t)a->post_weight |
                                (uintptr_t)a->post_bias | (uintptr_t)a->pre_weight | (uintptr_t)a->pre_bias | (uintptr_t)a->z;
    const uintptr_t stream_ptrs = (uintptr_t)a->x | (uintptr_t)a->h;
    KATZ_CHECK_ARG((half_ptrs & 1) == 0 && (stream_ptrs & (f32 ? 3 : 1)) == 0, KATZ_EALIGN);
    // 16-byte vectors where every row of every tensor starts on a 16-byte boundary, single elements otherwise
    const long long half_strides = a->y_sb | a->y_ss | a->z_sb | a->z_ss | a->gate_sb | a->gate_ss | a->scale_sb | a->scale_ss |
                                   a->shift_sb | a->shift_ss;
    const long long stream_strides = a->x_sb | a->x_ss | a->h_sb | a->h_ss;
    const bool vec = a->C % 8 == 0 && ((half_ptrs | stream_ptrs) & 15) == 0 && (half_strides & 7) == 0 && (stream_strides & (f32 ? 3 : 7)) == 0;
    ResidualNormParams p{};
    p.x = a->x; p.y = (const __half*)a->y; p.gate = (const __half*)a->gate; p.scale = (const __half*)a->scale; p.shift = (const __half*)a->shift;
    p.post_w = (const __half*)a->post_weight; p.post_b = (const __half*)a->post_bias;
    p.pre_w = (const __half*)a->pre_weight; p.pre_b = (const __half*)a->pre_bias;
    p.h = a->h; p.z = (__half*)a->z;
    p.x_sb = a->x_sb; p.x_ss = a->x_ss; p.y_sb = a->y_sb; p.y_ss = a->y_ss; p.h_sb = a->h_sb; p.h_ss = a->h_ss; p.z_sb = a->z_sb;
    p.z_ss = a->z_ss; p.gate_sb = a->gate_sb; p.gate_ss = a->gate_ss; p.scale_sb = a->scale_sb; p.scale_ss = a->scale_ss;
    p.shift_sb = a->shift_sb; p.shift_ss = a->shift_ss;
    p.S = a->S; p.C = a->C; p.rows = rows;
    p.post_kind = a->post_kind; p.pre_kind = a->pre_kind; p.post_eps = a->post_eps; p.pre_eps = a->pre_eps;
    p.residual_scale = a->residual_scale;
    if (vec) dispatch_residual_norm<true>(p, f32, (cudaStream_t)stream);
    else dispatch_residual_norm<false>(p, f32, (cudaStream_t)stream);
    KATZ_LAUNCH_RET();
}
