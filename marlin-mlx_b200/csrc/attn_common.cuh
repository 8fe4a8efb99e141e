// attn_common.cuh — device helpers of the attention kernels over the quantized cache.
#pragma once

#include "common.cuh"
#include "kv_cache.cuh"

namespace marlin {

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// bf16x2 of (lo, hi), each rounded to nearest even
__device__ __forceinline__ uint32_t bf16x2_of(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}

__device__ __forceinline__ uint32_t bf16x2_min(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("min.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

constexpr uint32_t kBf16One2 = 0x3F803F80u, kBf16Neg128x2 = 0xC300C300u, kBf16Half2 = 0x3F003F00u,
                   kBf16Magic = 0x43004300u, kBf16NegZero2 = 0x80008000u;

// Two 4-bit codes at bits [0,4) and [16,20) of w -> bf16x2 s q + b.  OR-ing the exponent of 128 gives
// 128 + q exactly, one FMA removes the 128 (exact), one forms q s + b with a single rounding.
__device__ __forceinline__ uint32_t dequant4(uint32_t w, uint32_t s2, uint32_t b2) {
    const uint32_t v = lop3_and_or(w, 0x000F000Fu, kBf16Magic);
    return bf16x2_fma(bf16x2_fma(v, kBf16One2, kBf16Neg128x2), s2, b2);
}
// Two 8-bit codes at bits [0,8) and [16,24) of w -> bf16x2 s q + b.  bf16 keeps 7 fraction bits, so the
// OR gives v = 128 + q below 128 and v = 2 q from 128 on (bit 7 lands on the exponent): q is the smaller
// of v - 128 and v / 2 in both cases, every step exact.
__device__ __forceinline__ uint32_t dequant8(uint32_t w, uint32_t s2, uint32_t b2) {
    const uint32_t v = lop3_and_or(w, 0x00FF00FFu, kBf16Magic);
    const uint32_t q = bf16x2_min(bf16x2_fma(v, kBf16One2, kBf16Neg128x2), bf16x2_fma(v, kBf16Half2, kBf16NegZero2));
    return bf16x2_fma(q, s2, b2);
}

// The tokens [q0, q0 + n) and cached positions of sequence b, made safe: starts clamped to the tokens,
// at most max_q of them, lengths clamped to what the table can hold.  What had to be cut is recorded.
struct SeqSpan {
    int q0, n, len;
};
__device__ __forceinline__ SeqSpan seq_span(const AttnArgs& a, int b) {
    SeqSpan s;
    int q1;
    if (a.cu_q) {
        s.q0 = a.cu_q[b];
        q1 = a.cu_q[b + 1];
    } else {
        s.q0 = b;
        q1 = b + 1;
    }
    s.len = a.kv_lens[b];
    const int64_t cap = (int64_t)a.table_width * a.pool.page_units * kKvRows;
    bool bad = s.q0 < 0 || q1 < s.q0 || q1 > a.tokens || s.len < 0 || s.len > cap;
    s.q0 = min(max(s.q0, 0), (int)a.tokens);
    s.n = min(max(q1, s.q0), (int)a.tokens) - s.q0;
    if (s.n > a.max_q) {
        s.n = a.max_q;
        bad = true;
    }
    s.len = (int)min((int64_t)max(s.len, 0), cap);
    if (bad) record_device_error(kDevErrBadIndex);
    return s;
}

// Page of the cache behind entry i of sequence b's table row; an index outside the pool is recorded and
// reads page 0.
__device__ __forceinline__ int table_page(const AttnArgs& a, int b, int i) {
    int p = a.table[(int64_t)b * a.table_stride + i];
    if (p < 0 || p >= a.pool.pages) {
        record_device_error(kDevErrBadIndex);
        p = 0;
    }
    return p;
}

}  // namespace marlin
