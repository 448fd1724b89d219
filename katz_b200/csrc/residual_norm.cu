// The norms after and before a block, with the block's gate and the residual scale between them, in one pass:
//   u = post(y)                    (LayerNorm, RMSNorm or none; y: the block's output)
//   h = residual_scale * x + gate * u
//   z = pre(h) * (1 + scale) + shift   (LayerNorm, RMSNorm or none: the next block's input)
// LayerNorm(v) = (v - mean) / sqrt(var + eps) * weight + bias, RMSNorm(v) = v / sqrt(mean of v^2 + eps) * weight + bias; weight and
// bias are optional, gate, scale and shift may be per channel, per sample or per token (strides of zero).
//
// Bound by HBM: x and y are read once, h and z written once, 8 bytes per element in fp16; next by instructions, so the
// arithmetic is packed (two fp32 lanes an instruction). A row stays in registers from the load to the store; statistics are
// fp32, of the values before any rounding (z is computed from the unrounded h), and the variance is the mean of squared
// differences from the mean, so a row whose mean is large loses nothing. Rows of up to 1280 channels belong to one warp (sums
// by shuffles, no barrier), longer ones to 4 or 16 warps. Measured: 32768 rows of 640 channels with an fp32 stream 44.5 us for
// 252 MB (5.7 TB/s), 2048 x 1280 with gate, scale and shift 4.7 us (21 MB).
#include "tc05.cuh"      // packed fp32 arithmetic

namespace katz {

using tc05::add2;
using tc05::fma2;
using tc05::mul2;

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

// A thread holds NU vectors of E consecutive channels, as pairs: eight (16 bytes of fp16) beside an fp16 stream, four beside an
// fp32 one, so that a warp's accesses to either are contiguous. Channels past the last hold zeros; FULL: there are none.
template <int T, int E, bool VEC>
__device__ __forceinline__ int channel(int i, int e, int tid) {      // of element e of vector i
    return VEC ? (i * T + tid) * E + e : (i * E + e) * T + tid;
}

__device__ __forceinline__ void load_vector(const __half* p, float2 (&v)[4]) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    v[0] = unpack_half2(w.x), v[1] = unpack_half2(w.y), v[2] = unpack_half2(w.z), v[3] = unpack_half2(w.w);
}
__device__ __forceinline__ void load_vector(const __half* p, float2 (&v)[2]) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    v[0] = unpack_half2(w.x), v[1] = unpack_half2(w.y);
}
__device__ __forceinline__ void load_vector(const float* p, float2 (&v)[2]) {
    const float4 w = *reinterpret_cast<const float4*>(p);
    v[0] = make_float2(w.x, w.y), v[1] = make_float2(w.z, w.w);
}
__device__ __forceinline__ uint32_t pack(float2 v) { return pack_half2(v.x, v.y); }
__device__ __forceinline__ void store_vector(__half* p, const float2 (&v)[4]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack(v[0]), pack(v[1]), pack(v[2]), pack(v[3]));
}
__device__ __forceinline__ void store_vector(__half* p, const float2 (&v)[2]) { *reinterpret_cast<uint2*>(p) = make_uint2(pack(v[0]), pack(v[1])); }
__device__ __forceinline__ void store_vector(float* p, const float2 (&v)[2]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
}

template <int T_, int NU_, int E_, bool VEC_, bool FULL_>
struct RowOf {
    static constexpr int T = T_, NU = NU_, E = E_;
    static constexpr bool VEC = VEC_, FULL = FULL_;
    float2 v[NU][E / 2];

    static __device__ __forceinline__ bool in(int i, int tid, int C) { return FULL || channel<T, E, VEC>(i, 0, tid) < C; }      // VEC
    template <typename F>
    __device__ __forceinline__ void each(F f) {
#pragma unroll
        for (int i = 0; i < NU; ++i)
#pragma unroll
            for (int e = 0; e < E / 2; ++e) v[i][e] = f(v[i][e], i, e);
    }
    template <typename S>
    __device__ __forceinline__ void load(const S* src, int C, int tid) {
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            if constexpr (!FULL) {
#pragma unroll
                for (int e = 0; e < E / 2; ++e) v[i][e] = make_float2(0.f, 0.f);
            }
            if constexpr (VEC) {
                if (in(i, tid, C)) load_vector(src + channel<T, E, VEC>(i, 0, tid), v[i]);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int c = channel<T, E, VEC>(i, e, tid);
                    if (c < C) (e & 1 ? v[i][e / 2].y : v[i][e / 2].x) = (float)src[c];
                }
            }
        }
    }
    template <typename S>
    __device__ __forceinline__ void store(S* dst, int C, int tid) const {
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            if constexpr (VEC) {
                if (in(i, tid, C)) store_vector(dst + channel<T, E, VEC>(i, 0, tid), v[i]);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int c = channel<T, E, VEC>(i, e, tid);
                    if (c < C) dst[c] = (S)(e & 1 ? v[i][e / 2].y : v[i][e / 2].x);
                }
            }
        }
    }
    // v <- normalised v (weight and bias applied)
    __device__ __forceinline__ void normalise(int kind, const __half* weight, const __half* bias, float eps, int C, int tid, float* red,
                                              int& slot) {
        const float inv_c = 1.0f / (float)C;
        if (kind == KATZ_NORM_LAYER) {
            float2 s = make_float2(0.f, 0.f);
            each([&](float2 a, int, int) { s = add2(s, a); return a; });
            const float mean = row_sum<T>(s.x + s.y, red, slot) * inv_c;
            const float2 m = make_float2(-mean, -mean);
            each([&](float2 a, int i, int e) {
                float2 d = add2(a, m);
                if constexpr (!FULL) {      // what lies past the last channel stays zero
                    if (channel<T, E, VEC>(i, 2 * e, tid) >= C) d.x = 0.f;
                    if (channel<T, E, VEC>(i, 2 * e + 1, tid) >= C) d.y = 0.f;
                }
                return d;
            });
        }
        float2 q = make_float2(0.f, 0.f);
        each([&](float2 a, int, int) { q = fma2(a, a, q); return a; });
        const float rstd = rsqrtf(row_sum<T>(q.x + q.y, red, slot) * inv_c + eps);
        const float2 r = make_float2(rstd, rstd);
        each([&](float2 a, int, int) { return mul2(a, r); });
        if (weight) {
            RowOf g;
            g.load(weight, C, tid);
            each([&](float2 a, int i, int e) { return mul2(a, g.v[i][e]); });
        }
        if (bias) {
            RowOf b;
            b.load(bias, C, tid);
            each([&](float2 a, int i, int e) { return add2(a, b.v[i][e]); });
        }
    }
};

// one row per T threads; a CTA of max(T, 128) threads
template <int T, int NU, bool VEC, bool F32, bool FULL>
__global__ void __launch_bounds__(T > 128 ? T : 128) residual_norm_kernel(const ResidualNormParams p) {
    typedef typename Stream<F32>::T XT;
    typedef RowOf<T, NU, F32 ? 4 : 8, VEC, FULL> Row;
    __shared__ float red[2 * (T > 32 ? T / 32 : 1)];
    constexpr int ROWS = T >= 128 ? 1 : 128 / T;
    pdl_wait();
    pdl_launch_dependents();
    const int tid = threadIdx.x % T;
    const uint32_t row = blockIdx.x * ROWS + threadIdx.x / T;
    if (row >= (uint32_t)p.rows) return;      // uniform over the threads of a row
    const uint32_t b = row / (uint32_t)p.S, s = row - b * p.S;
    int slot = 0;
    Row h;
    h.load(static_cast<const XT*>(p.x) + b * p.x_sb + s * p.x_ss, p.C, tid);
    const float2 scale = make_float2(p.residual_scale, p.residual_scale);
    if (p.y) {
        Row u;
        u.load(p.y + b * p.y_sb + s * p.y_ss, p.C, tid);
        if (p.post_kind != KATZ_NORM_NONE) u.normalise(p.post_kind, p.post_w, p.post_b, p.post_eps, p.C, tid, red, slot);
        if (p.gate) {
            Row g;
            g.load(p.gate + b * p.gate_sb + s * p.gate_ss, p.C, tid);
            u.each([&](float2 a, int i, int e) { return mul2(a, g.v[i][e]); });
        }
        h.each([&](float2 a, int i, int e) { return fma2(scale, a, u.v[i][e]); });
    } else {
        h.each([&](float2 a, int, int) { return mul2(a, scale); });
    }
    if (p.h) h.store(static_cast<XT*>(p.h) + b * p.h_sb + s * p.h_ss, p.C, tid);
    if (p.pre_kind == KATZ_NORM_NONE) return;
    h.normalise(p.pre_kind, p.pre_w, p.pre_b, p.pre_eps, p.C, tid, red, slot);
    if (p.scale) {
        Row g;
        g.load(p.scale + b * p.scale_sb + s * p.scale_ss, p.C, tid);
        h.each([&](float2 a, int i, int e) { return fma2(a, g.v[i][e], a); });
    }
    if (p.shift) {
        Row g;
        g.load(p.shift + b * p.shift_sb + s * p.shift_ss, p.C, tid);
        h.each([&](float2 a, int i, int e) { return add2(a, g.v[i][e]); });
    }
    h.store(p.z + b * p.z_sb + s * p.z_ss, p.C, tid);
}

template <int T, int NU, bool VEC, bool F32>
static void launch_residual_norm(const ResidualNormParams& p, cudaStream_t st) {
    constexpr int ROWS = T >= 128 ? 1 : 128 / T;
    const unsigned grid = (unsigned)ceil_div_ll(p.rows, ROWS);
    auto kernel = residual_norm_kernel<T, NU, VEC, F32, false>;
    if constexpr (VEC) {
        if (p.C == T * NU * (F32 ? 4 : 8)) kernel = residual_norm_kernel<T, NU, VEC, F32, true>;
    }
    launch_k(kernel, grid, T > 128 ? T : 128, 0, st, p);
}

// T threads of up to NU vectors: the fewest vectors that hold the row
template <int T, int NU, int MAX, bool VEC, bool F32>
static void pick_vectors(const ResidualNormParams& p, cudaStream_t st) {
    if constexpr (NU < MAX) {
        if (p.C > T * NU * (F32 ? 4 : 8)) return pick_vectors<T, NU + 1, MAX, VEC, F32>(p, st);
    }
    launch_residual_norm<T, NU, VEC, F32>(p, st);
}

template <bool VEC, bool F32>
static void dispatch_residual_norm(const ResidualNormParams& p, cudaStream_t st) {
    constexpr int E = F32 ? 4 : 8, MORE = F32 ? 2 : 1;
    if constexpr (!VEC) {      // single elements: a few sizes
        if (p.C <= 32 * 16) launch_residual_norm<32, 2 * MORE, VEC, F32>(p, st);
        else if (p.C <= 128 * 16) launch_residual_norm<128, 2 * MORE, VEC, F32>(p, st);
        else launch_residual_norm<512, 4 * MORE, VEC, F32>(p, st);
    } else if (p.C <= 32 * 5 * MORE * E) {
        pick_vectors<32, 1, 5 * MORE, VEC, F32>(p, st);
    } else if (p.C <= 128 * 4 * MORE * E) {
        pick_vectors<128, 2 * MORE, 4 * MORE, VEC, F32>(p, st);
    } else {
        pick_vectors<512, 2 * MORE, 4 * MORE, VEC, F32>(p, st);
    }
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
    cudaStream_t st = (cudaStream_t)stream;
    if (f32) vec ? dispatch_residual_norm<true, true>(p, st) : dispatch_residual_norm<false, true>(p, st);
    else vec ? dispatch_residual_norm<true, false>(p, st) : dispatch_residual_norm<false, false>(p, st);
    KATZ_LAUNCH_RET();
}
