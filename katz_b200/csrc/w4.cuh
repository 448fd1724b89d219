// The 4-bit weight format, shared by the kernels that make it, read it back and multiply with it.
//
// A weight matrix [N, K] (K a multiple of 32) is held as codes q[N, K/2] (one byte per two weights, the even k in the low
// four bits), bf16 scales [N, J] and, optionally, zero points [N, J] (0..15, one byte each; 8 without them) for J = ceil(K /
// group) groups of 32, 64 or 128 consecutive k, the last of which may be short: w = scale * (code - zero).
//
// A bf16 scale has 8 significant bits and code - 8 needs at most 3 (8 itself is a power of two), so the product is exact in
// fp16 and the tensor cores multiply with the weight itself, without a rounding between the format and the product. With
// zero points |code - zero| reaches 15: the odd ones above 8 round in the 12th bit.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"

namespace katz {
namespace w4 {

// The products take 64 * weight as their fp16 operand and undo the factor in fp32 at the end: scales from 2^-23 (fp16's
// smallest subnormal step times 64, still exact) to 68 (15 * 64 * 68 stays below fp16's largest value) are covered, instead
// of 2^-17 to 4366, and weights of 1e-5 keep their bits.
constexpr float OPERAND_SCALE = 64.0f, OPERAND_UNSCALE = 1.0f / 64.0f;

__device__ __forceinline__ float bf16_bits_to_float(unsigned short b) { return __uint_as_float((uint32_t)b << 16); }
__device__ __forceinline__ __half2 as_half2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

// (w & mask) | 0x64006400 in one three-input logic instruction
template <uint32_t MASK>
__device__ __forceinline__ uint32_t and_or_1024(uint32_t w) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "n"(MASK), "r"(0x64006400u));
    return r;
}

// One word (8 codes, k = 0..7) -> code - zero as four fp16 pairs (k0,k4), (k1,k5), (k2,k6), (k3,k7):
//   (word & 0x000f000f) | 0x6400'6400 is the pair (1024 + c0, 1024 + c4) in fp16: subtracting 1024 + zero is exact;
//   (word & 0x00f000f0) | 0x6400'6400 is (1024 + 16 c1, 1024 + 16 c5): times 1/16, minus 64 + zero, is exact too.
__device__ __forceinline__ void unpack8(uint32_t w, __half2 low, __half2 high, __half2* d) {
    const __half2 sixteenth = __float2half2_rn(0.0625f);
    const uint32_t v = w >> 8;
    d[0] = __hadd2(as_half2(and_or_1024<0x000f000fu>(w)), low);
    d[1] = __hfma2(as_half2(and_or_1024<0x00f000f0u>(w)), sixteenth, high);
    d[2] = __hadd2(as_half2(and_or_1024<0x000f000fu>(v)), low);
    d[3] = __hfma2(as_half2(and_or_1024<0x00f000f0u>(v)), sixteenth, high);
}
// 16 bytes of shared memory by 32-bit address
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}

}  // namespace w4

struct W4Params {
    const __half* x;
    const unsigned char* q;
    const unsigned short* scale;
    const unsigned char* zero;
    const __half* bias;
    const __half* residual;
    __half* out;
    long long ldx, ldo, ldr;
    int M, N, K, J, group_shift;
    int act;
    float out_scale;
};

// The product for more rows on the tcgen05 path (w4_tc05.cu): p.x 16-byte aligned with ldx % 8 == 0, K >= W4_TC05_MIN_K.
constexpr int W4_TC05_MIN_K = 128;
int linear_w4_tc05(const W4Params& p, cudaStream_t st);

}  // namespace katz
