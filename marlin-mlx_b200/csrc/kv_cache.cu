// kv_cache.cu — what a decoder's attention layer does between its projections and its attention:
// the norms of the query and key heads with the position rotation in one pass, the quantizing write
// of keys and values into the paged cache, and the read back.  All three are bound by bytes (large
// calls) or by one launch (a decode step).
#include "kv_cache.cuh"

#include <algorithm>

#include "common.cuh"
#include "q4_host.cuh"
#include "q4_misc.cuh"

namespace marlin {
namespace {

// 8 consecutive elements as binary32
__device__ __forceinline__ void load8(const void* base, int64_t elt, bool bf16, float v[8]) {
    if (bf16) {
        const uint4 r = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + elt);
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    } else {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + elt);
        const float4 a = p[0], b = p[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    }
}

__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}

// ------------------------------------------------------------------------------------------------
// Head norms and rotation.  Per token t and head row x[dim]:
//   n = x * rsqrt(mean(x^2) + eps) * (1 + w)           (the offset weights of rms_norm)
//   (a, b) -> (a cos - b sin, b cos + a sin)            for the rot/2 pairs of the first rot features,
//   angle = position[axis of the pair][t] * freq        pairs (i, i + rot/2) or (2i, 2i + 1).
// One CTA per token: the rot/2 sines and cosines are formed once in shared memory (the angle in
// binary64 and reduced by whole turns, since a position near 10^6 leaves binary32 no fraction), then
// dim/8 lanes take a head row, 8 features each, sums and products in binary32, one rounding at the
// store.  The half layout's partner features sit in another lane of the same row (rot % 16 == 0), so
// they come by shuffle.
// ------------------------------------------------------------------------------------------------
template <int D, bool BF16_IN, bool BF16_OUT>
__global__ void __launch_bounds__(1024) qk_norm_rope_kernel(const __grid_constant__ RopeArgs a) {
    constexpr int LANES = D / 8;
    __shared__ float2 cs[128];
    const int64_t t = blockIdx.x;
    const int tid = threadIdx.x, sub = tid & (LANES - 1);
    pdl_wait();
    pdl_launch_dependents();
    for (int i = tid; i < a.rot / 2; i += blockDim.x) {
        const int ax = (a.axis[i >> 4] >> ((i & 15) * 2)) & 3;
        const double ang = (double)a.positions[(int64_t)ax * a.tokens + t] * (double)a.freqs[i];
        const double turns = rint(ang * 0.15915494309189535);
        float s, c;
        sincosf((float)fma(-turns, 6.283185307179586, ang), &s, &c);
        cs[i] = make_float2(c, s);
    }
    float w[2][8];
    load8(a.qw, sub * 8, true, w[0]);
    load8(a.kw, sub * 8, true, w[1]);
    __syncthreads();
    const int rows = a.heads + a.kv_heads, half = a.rot / 2;
    const int per_pass = blockDim.x / LANES;
    for (int r0 = 0; r0 < rows; r0 += per_pass) {
        const int row = r0 + tid / LANES;
        const bool live = row < rows;
        const bool isk = row >= a.heads;
        const int head = isk ? row - a.heads : row;
        float v[8] = {};
        if (live) {
            if (isk)
                load8(a.k, t * a.k_ts + head * a.k_hs + sub * 8, BF16_IN, v);
            else
                load8(a.q, t * a.q_ts + head * a.q_hs + sub * 8, BF16_IN, v);
        }
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fmaf(v[i], v[i], sum);
#pragma unroll
        for (int o = 1; o < LANES; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const float rs = rsqrtf(sum * (1.0f / D) + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= rs * (1.0f + w[isk][i]);
        const int d0 = sub * 8;
        if (a.interleaved) {
            if (d0 < a.rot) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 e = cs[d0 / 2 + i];
                    const float x = v[2 * i], y = v[2 * i + 1];
                    v[2 * i] = x * e.x - y * e.y;
                    v[2 * i + 1] = y * e.x + x * e.y;
                }
            }
        } else {
            const bool first = d0 < half, turn = d0 < a.rot;
            const int src = (tid & 31) + (turn ? (first ? half / 8 : -half / 8) : 0);
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = __shfl_sync(0xffffffffu, v[i], src);
            if (turn) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 e = cs[first ? d0 + i : d0 + i - half];
                    v[i] = v[i] * e.x + (first ? -p[i] : p[i]) * e.y;
                }
            }
        }
        if (!live) continue;
        void* base = isk ? a.k_out : a.q_out;
        const int64_t o = (t * (isk ? a.kv_heads : a.heads) + head) * D + d0;
        if (BF16_OUT) {
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + o) =
                make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
        } else {
            float4* y = reinterpret_cast<float4*>(static_cast<float*>(base) + o);
            y[0] = make_float4(v[0], v[1], v[2], v[3]);
            y[1] = make_float4(v[4], v[5], v[6], v[7]);
        }
    }
}

// ------------------------------------------------------------------------------------------------
// Quantizing write.  Eight lanes take one group of 64 features of one (token, head, key or value):
// the rule of quantize_kernel (binary32, no contraction, ties away from zero) with 15 or 255 steps on
// the values rounded to bf16, so a row of the cache holds exactly what marlin_q4_quantize makes of it.
// A lane's eight codes are one (4 bits) or two (8 bits) words of the unit.  Slots below zero are
// skipped; a slot outside the pool is skipped and recorded.
// ------------------------------------------------------------------------------------------------
template <int BITS, bool BF16_IN>
__global__ void __launch_bounds__(256) kv_write_kernel(KvPool c, const void* __restrict__ k, int64_t k_ts, int64_t k_hs,
                                                       const void* __restrict__ v, int64_t v_ts, int64_t v_hs,
                                                       const int32_t* __restrict__ slots, int64_t items) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane8 = threadIdx.x & 7;
    const int64_t item = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 3;
    const int groups = c.dim / 64, rb = c.dim * BITS / 8;
    const bool valid = item < items;
    // item = ((token * kv_heads + head) * 2 + value) * groups + group
    const int64_t i2 = valid ? item / groups : 0;
    const int g = valid ? (int)(item - i2 * groups) : 0;
    const bool isv = i2 & 1;
    const int64_t th = i2 >> 1, t = th / c.kv_heads;
    const int h = (int)(th - t * c.kv_heads);
    const int64_t slot = valid ? slots[t] : -1;
    const int64_t unit = slot / kKvRows;
    bool put = slot >= 0;
    if (put && unit >= c.pages * c.page_units) {
        put = false;
        if (lane8 == 0) record_device_error(kDevErrBadIndex);
    }
    float x[8] = {};
    if (put) {
        if (isv)
            load8(v, t * v_ts + h * v_hs + g * 64 + lane8 * 8, BF16_IN, x);
        else
            load8(k, t * k_ts + h * k_hs + g * 64 + lane8 * 8, BF16_IN, x);
    }
    float lo = INFINITY, hi = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (!BF16_IN) x[i] = bf16_round(x[i]);
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    constexpr float kTop = (float)((1 << BITS) - 1);
    float scale = fmaxf(__fdiv_rn(__fsub_rn(hi, lo), kTop), 1e-7f);
    const bool side = fabsf(lo) > fabsf(hi);
    scale = side ? scale : -scale;
    const float edge = side ? lo : hi;
    const float steps = roundf(__fdiv_rn(edge, scale));
    float bias = 0.0f;
    if (steps != 0.0f) {
        scale = __fdiv_rn(edge, steps);
        bias = edge;
    }
    uint32_t code[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        code[i] = (uint32_t)fminf(fmaxf(roundf(__fdiv_rn(__fsub_rn(x[i], bias), scale)), 0.0f), kTop);
    if (!put) return;
    const int r = (int)(slot % kKvRows);
    const int64_t page = unit / c.page_units;
    uint8_t* u = c.data + ((page * c.kv_heads + h) * c.page_units + unit % c.page_units) * (int64_t)(32 * (rb + 4 * groups));
    const int j = (g * 64 + lane8 * 8) * BITS / 8;
    uint8_t* dst = u + (isv ? kv_value_code(r, j, rb, groups) : kv_key_code(r, j, rb));
    if (BITS == 4) {
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) word |= code[i] << (4 * i);
        *reinterpret_cast<uint32_t*>(dst) = word;
    } else {
        *reinterpret_cast<uint2*>(dst) = make_uint2(code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24,
                                                    code[4] | code[5] << 8 | code[6] << 16 | code[7] << 24);
    }
    if (lane8 == 0)
        *reinterpret_cast<uint32_t*>(u + (isv ? kv_value_pair(r, g, rb, groups) : kv_key_pair(r, g, rb, groups))) =
            f32_to_bf16_bits(scale) | (f32_to_bf16_bits(bias) << 16);
}

// Read back: eight features per thread, bf16(scale * code + bias) with one rounding of the exact value
// (the operand of the attention kernels).  Rows of slots below zero read as zero, as do rows of slots
// outside the pool, which are recorded.
template <int BITS>
__global__ void __launch_bounds__(256) kv_read_kernel(KvPool c, const int32_t* __restrict__ slots, int64_t items,
                                                      uint16_t* __restrict__ ko, uint16_t* __restrict__ vo) {
    pdl_wait();
    pdl_launch_dependents();
    const int64_t item = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (item >= items) return;
    const int groups = c.dim / 64, rb = c.dim * BITS / 8, chunks = c.dim / 8;
    // item = ((token * kv_heads + head) * 2 + value) * chunks + chunk
    const int64_t i2 = item / chunks;
    const int ch = (int)(item - i2 * chunks);
    const bool isv = i2 & 1;
    const int64_t th = i2 >> 1, t = th / c.kv_heads;
    const int h = (int)(th - t * c.kv_heads);
    const int64_t slot = slots[t], unit = slot / kKvRows;
    uint4 o = make_uint4(0u, 0u, 0u, 0u);
    if (slot >= 0 && unit < c.pages * c.page_units) {
        const int r = (int)(slot % kKvRows), g = ch / 8, j = ch * BITS;
        const int64_t page = unit / c.page_units;
        const uint8_t* u =
            c.data + ((page * c.kv_heads + h) * c.page_units + unit % c.page_units) * (int64_t)(32 * (rb + 4 * groups));
        const uint8_t* src = u + (isv ? kv_value_code(r, j, rb, groups) : kv_key_code(r, j, rb));
        const uint32_t pair = *reinterpret_cast<const uint32_t*>(
            u + (isv ? kv_value_pair(r, g, rb, groups) : kv_key_pair(r, g, rb, groups)));
        const uint32_t s2 = __byte_perm(pair, 0, 0x1010), b2 = __byte_perm(pair, 0, 0x3232);
        if (BITS == 4) {
            o = dequant_word(*reinterpret_cast<const uint32_t*>(src), s2, b2);
        } else {
            const uint2 w = *reinterpret_cast<const uint2*>(src);
            // codes up to 255 are exact in bf16, so one bf16 FMA rounds the exact value once
            uint32_t p[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t q = i < 2 ? w.x : w.y;
                const uint32_t two = pack_bf16x2((float)((q >> (16 * (i & 1))) & 255u), (float)((q >> (16 * (i & 1) + 8)) & 255u));
                p[i] = bf16x2_fma(two, s2, b2);
            }
            o = make_uint4(p[0], p[1], p[2], p[3]);
        }
    } else if (slot >= 0) {
        record_device_error(kDevErrBadIndex);
    }
    *reinterpret_cast<uint4*>((isv ? vo : ko) + (th * c.dim + ch * 8)) = o;
}

template <typename... P, typename... A>
cudaError_t launch_pdl(void (*kernel)(P...), int64_t blocks, int threads, bool pdl, cudaStream_t stream, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

template <int D>
cudaError_t rope_dim(const RopeArgs& a, bool bi, bool bo, int64_t blocks, int threads, bool pdl, cudaStream_t s) {
    if (bi && bo) return launch_pdl(qk_norm_rope_kernel<D, true, true>, blocks, threads, pdl, s, a);
    if (bi) return launch_pdl(qk_norm_rope_kernel<D, true, false>, blocks, threads, pdl, s, a);
    if (bo) return launch_pdl(qk_norm_rope_kernel<D, false, true>, blocks, threads, pdl, s, a);
    return launch_pdl(qk_norm_rope_kernel<D, false, false>, blocks, threads, pdl, s, a);
}

}  // namespace

cudaError_t launch_qk_norm_rope(const RopeArgs& a, int dtype, int out_dtype, bool pdl, cudaStream_t stream) {
    // few tokens: the whole token in one pass of its CTA; many: smaller CTAs, several per SM
    const int lanes = (a.heads + a.kv_heads) * (a.dim / 8);
    const int most = a.tokens <= 2 * device_num_sms() ? 1024 : 256;
    const int threads = std::min(most, (lanes + 31) / 32 * 32);
    const bool bi = dtype == kDtypeBF16, bo = out_dtype == kDtypeBF16;
    if (a.dim == 64) return rope_dim<64>(a, bi, bo, a.tokens, threads, pdl, stream);
    if (a.dim == 128) return rope_dim<128>(a, bi, bo, a.tokens, threads, pdl, stream);
    return rope_dim<256>(a, bi, bo, a.tokens, threads, pdl, stream);
}

cudaError_t launch_kv_write(const KvPool& c, const void* k, int64_t k_ts, int64_t k_hs, const void* v, int64_t v_ts,
                            int64_t v_hs, int dtype, const int32_t* slots, int64_t tokens, bool pdl, cudaStream_t stream) {
    const int64_t items = tokens * c.kv_heads * 2 * (c.dim / 64), blocks = (items * 8 + 255) / 256;
    const bool b = dtype == kDtypeBF16;
    auto go = [&](auto kernel) {
        return launch_pdl(kernel, blocks, 256, pdl, stream, c, k, k_ts, k_hs, v, v_ts, v_hs, slots, items);
    };
    if (c.bits == 4) return b ? go(kv_write_kernel<4, true>) : go(kv_write_kernel<4, false>);
    return b ? go(kv_write_kernel<8, true>) : go(kv_write_kernel<8, false>);
}

cudaError_t launch_kv_read(const KvPool& c, const int32_t* slots, int64_t tokens, uint16_t* k, uint16_t* v, bool pdl,
                           cudaStream_t stream) {
    const int64_t items = tokens * c.kv_heads * 2 * (c.dim / 8), blocks = (items + 255) / 256;
    if (c.bits == 4) return launch_pdl(kv_read_kernel<4>, blocks, 256, pdl, stream, c, slots, items, k, v);
    return launch_pdl(kv_read_kernel<8>, blocks, 256, pdl, stream, c, slots, items, k, v);
}

int kv_device_error(bool clear) { return tu_device_error(clear); }

}  // namespace marlin
