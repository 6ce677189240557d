// What the kernels of the shared-prefix attention have in common: the two caches of a call, the partial results, and the
// conversion of stored codes.
#pragma once

#include "izb_common.cuh"

namespace izb {
namespace shared_prefix {

// One of the two caches of a call: rows of a page table with their lengths.
struct Source {
    const uint8_t* k;
    const uint8_t* v;
    const float* k_scales;
    const float* v_scales;
    const int* table;
    const int* lens;
    long long max_pages;
    int quant, page_size;
    int max_len;     // lengths on the device are cut to this
    int chunk;       // tokens per item
    int n_chunks;    // partial results a row can have from this cache
    int step_pages, step_rest;  // 128 tokens in pages and what is left of them
};

struct Params {
    Source prefix, own;
    const __nv_bfloat16* q;
    float* acc;       // [rows][chunks][D], rows = batch * heads
    float2* ml;       // [rows][chunks]: maximum (log2 scale) and sum
    long long ld_q;
    int seqs, heads, kv_heads, g;  // sequences per group, query heads per KV head
    int row_blocks, prefix_items;
    int cluster_rows;              // a cluster's items: where in shared memory their rows' results lie
    int* status;
    uint32_t q_sign;   // flips q where the scale is negative, so that the largest product is the largest score
    float scale_log2;  // |scale| / ln 2
    float margin;      // 8 / scale_log2: a growth of 2^8 in weight, in units of the products
};

__device__ __forceinline__ int length_of(const Source& s, int row) { return min(max(s.lens[row], 0), s.max_len); }

// `n` of the 16 (4) bytes come from src, the rest is zero
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int n) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, int n) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Codes -> bf16x2.  (x & mask) | base takes one instruction when both constants are in registers and two when they are
// immediates, so they are put there once, out of the compiler's sight.
template <int Q>
struct CodeBits {
    uint32_t mask, base, top, bias;
    __device__ __forceinline__ CodeBits() {
        if (Q == IZB_KV_INT8) {
            asm volatile("mov.b32 %0, 0x007F007F;\n\tmov.b32 %1, 0x00800080;\n\tmov.b32 %2, 0xC300C300;" : "=r"(mask), "=r"(top), "=r"(bias));
        } else {
            asm volatile("mov.b32 %0, 0x000F000F;\n\tmov.b32 %1, 0xC308C308;" : "=r"(mask), "=r"(bias));
            top = 0u;
        }
        asm volatile("mov.b32 %0, 0x43004300;" : "=r"(base));
    }
    // Two codes in the low bits of the halves of x, exact.  Int8 (code = byte - 128): 128 + (byte & 127) is the bf16 0x4300 |
    // low bits; what is left to add is -256 for bytes below 128 and -128 above.  Q4_0 (code = nibble - 8): 128 + nibble - 136.
    __device__ __forceinline__ uint32_t pair(uint32_t x) const {
        const uint32_t low = lop3<0xEA>(x, mask, base);                                     // (x & mask) | base
        return hfma2(low, 0x3F803F80u, Q == IZB_KV_INT8 ? lop3<0xAE>(x, top, bias) : bias);  // (~x & top) | bias
    }
};
// code * scale rounded to bf16 as the stored value is defined.  The fp32 scale enters as two bf16 parts; the small
// part, 2^-8 of it at most, and its product are rounded to 8 bits each, so the sum's one rounding sees the product to 2^-15.
__device__ __forceinline__ uint32_t q4_value(uint32_t code2, uint32_t hi2, uint32_t lo2) { return hfma2(code2, hi2, hmul2(code2, lo2)); }
// the two parts of two scales side by side
__device__ __forceinline__ void split_scales(float a, float b, uint32_t& hi2, uint32_t& lo2) {
    hi2 = pack_bf16x2(a, b);
    lo2 = pack_bf16x2(a - bf16_lo_to_f32(hi2), b - bf16_hi_to_f32(hi2));
}

// The tensor-memory kernel (shared_prefix_tc.cu): partial results of the prefix, in blocks of 128 query rows, or of 256
// where there are more than 128.
constexpr int TC_ROWS = 128;
int launch_prefix_tc(izb_ctx* ctx, cudaStream_t s, const Params& p, int head_dim, int64_t groups);

}  // namespace shared_prefix
}  // namespace izb
