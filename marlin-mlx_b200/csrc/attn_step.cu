// attn_step.cu — attention of few query rows over the paged, quantized cache: decode steps and short
// runs of new tokens.
//
// Rows are the (token, head of the group) pairs of one kv head, 8 or 16 to a tile.  Per tile and 16
// cached positions, with K and V dequantized in registers (bf16, one rounding of the exact value):
//   S^T[16 x rows] = K Q^T          mma m16n8k16, A = K from the codes, B = Q
//   P = 2^(S scale log2e - m)       running maximum m and sum l per row, binary32
//   O^T[dim x rows] += V^T P^T      A = V^T from the codes, B = P^T (one 8x8 transpose of the bf16 pairs)
// Taking the positions (then the features) as the M side lets 8 rows fill an MMA, so a decode step of
// up to 8 heads per kv head wastes none of the dequantized operand.
//
// Bound: bytes of the cache, or the issue slots of the dequantization (about 2 instructions per value
// at 4 bits).  Each warp owns a ring of units fed by bulk copies (one contiguous unit per copy) and
// takes every fourth pair of units of its CTA's range, with its own m, l and O; the four warps are
// joined once at the end of a range in shared memory.  The work of all tiles, in units, is laid end to
// end and cut into equal shares, one per CTA, so that lengths of any mix load the SMs evenly; a tile
// that several CTAs touched is joined by a second kernel from their partial rows, in a fixed order.
#include <algorithm>

#include "attn_common.cuh"
#include "q4_host.cuh"

namespace marlin {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kMinShare = 2 * kWarps;  // units: one pair per warp

template <int D, int BITS, int NT>
struct StepCfg {
    static constexpr int RB = kv_row_bytes(D, BITS), G = D / 64, UB = kv_unit_bytes(D, BITS);
    static constexpr int ROWS = 8 * NT;
    static constexpr int STEPS = D / 16;   // MMAs along the features
    static constexpr int PANELS = RB < 64 ? 1 : RB / 64;
    static constexpr int CTAS = NT == 2 ? (D == 256 ? 1 : D == 128 ? 2 : 4) : D == 256 ? (BITS == 4 ? 3 : 2) : D == 128 ? (BITS == 4 ? 4 : 3) : 5;
    static constexpr int RING = D == 256 ? 3 : D == 128 ? (BITS == 4 ? 4 : 3) : (BITS == 4 ? 6 : 4);
    static constexpr uint32_t RING_BYTES = kWarps * RING * UB;
    static constexpr uint32_t MERGE_BYTES = kWarps * ROWS * D * 4;
    static constexpr uint32_t OFF_Q = RING_BYTES > MERGE_BYTES ? RING_BYTES : MERGE_BYTES;
    static constexpr uint32_t OFF_ML = OFF_Q + NT * STEPS * 32 * 8;
    static constexpr uint32_t OFF_BAR = OFF_ML + kWarps * ROWS * 8;
    static constexpr uint32_t OFF_PRE = OFF_BAR + kWarps * RING * 8;
    static constexpr uint32_t SMEM = OFF_PRE + (kAttnMaxBatch + 1) * 4 + 64;
};

// Workspace: [kAttnMaxBatch + 1] u32 prefix of the work, share (u32), then per slot ROWS (m, l) pairs,
// then per slot [ROWS][D] partial rows.  Slots 2 c and 2 c + 1 belong to CTA c (its first range, its last).
struct StepWork {
    uint32_t* prefix;
    float2* ml;
    float* o;
};
constexpr size_t kStepHead = ((kAttnMaxBatch + 2) * 4 + 255) / 256 * 256;
__host__ __device__ inline StepWork step_work(float* part, int grid, int rows) {
    uint8_t* p = reinterpret_cast<uint8_t*>(part);
    StepWork w;
    w.prefix = reinterpret_cast<uint32_t*>(p);
    w.ml = reinterpret_cast<float2*>(p + kStepHead);
    w.o = reinterpret_cast<float*>(p + kStepHead + (size_t)2 * grid * rows * 8);
    return w;
}

__device__ __forceinline__ uint32_t seq_work(const AttnArgs& a, const SeqSpan& s, int rows) {
    const uint32_t tiles = (uint32_t)((s.n * a.group + rows - 1) / rows);
    return (uint32_t)a.pool.kv_heads * tiles * (uint32_t)((s.len + kKvRows - 1) / kKvRows);
}

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

template <int D, int BITS, int NT>
__global__ void __launch_bounds__(kThreads, StepCfg<D, BITS, NT>::CTAS) attn_step_kernel(const __grid_constant__ AttnArgs a) {
    using C = StepCfg<D, BITS, NT>;
    extern __shared__ __align__(128) uint8_t smem[];
    uint32_t* pre = reinterpret_cast<uint32_t*>(smem + C::OFF_PRE);
    uint2* qf = reinterpret_cast<uint2*>(smem + C::OFF_Q);       // [NT][STEPS][32]
    float2* ml = reinterpret_cast<float2*>(smem + C::OFF_ML);    // [warp][ROWS]
    float4* merge = reinterpret_cast<float4*>(smem);             // [warp][ROWS][D / 4], over the ring
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    uint8_t* ring = smem + warp * (C::RING * C::UB);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR) + warp * C::RING;
    __shared__ uint32_t wsum[kWarps];
    __shared__ int stop;

    if (tid == 0) stop = 0;
    if (lane == 0) {
        for (int i = 0; i < C::RING; ++i) mbar_init(&bars[i], 1);
        fence_mbar_init();
    }
    pdl_wait();
    pdl_launch_dependents();
    // prefix sums of the sequences' work, in units
    uint32_t base = 0;
    if (tid == 0) pre[0] = 0;
    for (int b0 = 0; b0 < a.batch; b0 += kThreads) {
        const int b = b0 + tid;
        uint32_t v = 0;
        if (b < a.batch) {
            const SeqSpan s = seq_span(a, b);
            v = seq_work(a, s, C::ROWS);
            if (s.len == 0 && b % gridDim.x == blockIdx.x)  // no position to attend to: zero rows
                for (int64_t i = 0; i < (int64_t)s.n * a.heads * D / 8; ++i)
                    reinterpret_cast<uint4*>(a.out + (int64_t)s.q0 * a.heads * D)[i] = make_uint4(0u, 0u, 0u, 0u);
        }
        uint32_t x = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 31) wsum[warp] = x;
        __syncthreads();
        uint32_t before = base, all = base;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += wsum[w];
            all += wsum[w];
        }
        if (b < a.batch) pre[b + 1] = before + x;
        base = all;
    }
    __syncthreads();
    const uint32_t total = base;
    const uint32_t share = max((uint32_t)kMinShare, (total + gridDim.x - 1) / gridDim.x);
    const StepWork work = step_work(a.part, gridDim.x, C::ROWS);
    if (blockIdx.x == 0) {
        for (int b = tid; b <= a.batch; b += kThreads) work.prefix[b] = pre[b];
        if (tid == 0) work.prefix[kAttnMaxBatch + 1] = share;
    }
    const uint64_t w_begin = (uint64_t)blockIdx.x * share;
    const uint32_t w_end = (uint32_t)min((uint64_t)total, w_begin + share);

    uint32_t done = 0;  // units this warp has consumed so far (ring position and phase)
    for (uint32_t w0 = (uint32_t)min(w_begin, (uint64_t)total); w0 < w_end;) {
        // the range's sequence, kv head, row tile and units
        int lo = 0, hi = a.batch - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (pre[mid] <= w0) lo = mid; else hi = mid - 1;
        }
        const int b = lo;
        const SeqSpan s = seq_span(a, b);
        const uint32_t nu = (uint32_t)((s.len + kKvRows - 1) / kKvRows);
        const uint32_t tiles = (uint32_t)((s.n * a.group + C::ROWS - 1) / C::ROWS);
        const uint32_t in = w0 - pre[b], ti = in / nu;
        const int u0 = (int)(in - ti * nu), h = (int)(ti / tiles), row0 = (int)(ti % tiles) * C::ROWS;
        const int u1 = (int)min((uint32_t)nu, (uint32_t)u0 + (w_end - w0));
        const bool whole = u0 == 0 && u1 == (int)nu;
        const int slot = 2 * (int)blockIdx.x + (w0 == (uint32_t)w_begin ? 0 : 1);
        w0 += (uint32_t)(u1 - u0);
        const int nrows = min(C::ROWS, s.n * a.group - row0);
        // row r sees the positions below len - n + token + 1
        const int last_seen = s.len - s.n + (row0 + nrows - 1) / a.group + 1;
        const int first_seen = s.len - s.n + row0 / a.group + 1;
        const int ue = min(u1, (max(last_seen, 0) + kKvRows - 1) / kKvRows);  // units beyond hold nothing seen

        // this warp's units: pairs warp, warp + 4, ... of [u0, ue)
        auto unit_of = [&](int k) { return u0 + 2 * (warp + kWarps * (k >> 1)) + (k & 1); };
        const int left = max(0, ue - u0);
        const int full = left / (2 * kWarps), rest = left % (2 * kWarps) - 2 * warp;
        const int mine = 2 * full + min(2, max(0, rest));
        int page = 0, issued = 0;
        auto issue = [&](int upto) {
            for (; issued < upto; ++issued) {
                if ((issued & 31) == 0) {  // the pages of the next 32 units, one per lane
                    const int k = issued + lane;
                    if (k < mine) page = table_page(a, b, unit_of(k) / a.pool.page_units);
                }
                const int64_t pg = __shfl_sync(0xffffffffu, page, issued & 31);
                if (lane == 0) {
                    const int u = unit_of(issued);
                    const uint32_t at = (done + issued) % C::RING;
                    const uint8_t* src = a.pool.data + ((pg * a.pool.kv_heads + h) * a.pool.page_units + u % a.pool.page_units) * (int64_t)C::UB;
                    mbar_arrive_expect_tx(&bars[at], C::UB);
                    tma_bulk_g2s(ring + at * C::UB, src, C::UB, &bars[at]);
                }
            }
        };
        issue(min(mine, C::RING));

        // Q as B fragments; feature order = the order in which the key codes unpack
        for (int i = tid; i < NT * C::STEPS * 32; i += kThreads) {
            const int ln = i & 31, st = (i >> 5) % C::STEPS, nt = (i >> 5) / C::STEPS;
            const int r = row0 + nt * 8 + (ln >> 2), tt = ln & 3;
            uint2 v = make_uint2(0u, 0u);
            if (nt * 8 + (ln >> 2) < nrows) {
                const uint16_t* q = a.q + (int64_t)(s.q0 + r / a.group) * a.q_ts + (int64_t)(h * a.group + r % a.group) * a.q_hs;
                if (BITS == 4) {
                    const int d = (C::RB < 64 ? tt * 16 + (st >> 1) * 8 : (st >> 3) * 128 + tt * 32 + ((st & 7) >> 1) * 8) + (st & 1) * 2;
                    v.x = q[d] | ((uint32_t)q[d + 4] << 16);
                    v.y = q[d + 1] | ((uint32_t)q[d + 5] << 16);
                } else {
                    const int d = (st >> 2) * 64 + tt * 16 + (st & 3) * 4;
                    v.x = q[d] | ((uint32_t)q[d + 2] << 16);
                    v.y = q[d + 1] | ((uint32_t)q[d + 3] << 16);
                }
            }
            qf[i] = v;
        }
        __syncthreads();

        float m[NT][2], l[NT][2], o[NT][D / 16][4];
        int lim[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                m[nt][x] = -INFINITY;
                l[nt][x] = 0.f;
                lim[nt][x] = min(s.len, s.len - s.n + (row0 + nt * 8 + 2 * t + x) / a.group + 1);
            }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < D / 16; ++j)
#pragma unroll
                for (int x = 0; x < 4; ++x) o[nt][j][x] = 0.f;

        bool ok = true;
        for (int k = 0; k < mine; k += 2) {
            const bool two = k + 1 < mine;
            float sc[2][NT][4];
            const uint8_t* up[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t at = (done + k + e) % C::RING;
                up[e] = ring + at * C::UB;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int x = 0; x < 4; ++x) sc[e][nt][x] = 0.f;
                if (e == 1 && !two) continue;
                ok = ok && mbar_wait(&bars[at], ((done + k + e) / C::RING) & 1);
                const uint8_t* u = up[e];
#pragma unroll
                for (int p = 0; p < C::PANELS; ++p) {
                    const int grp = BITS == 4 ? (C::RB < 64 ? 0 : (p * 128 + t * 32) / 64) : p;
                    const uint32_t k0 = *reinterpret_cast<const uint32_t*>(u + kv_key_pair(g, grp, C::RB, C::G));
                    const uint32_t k1 = *reinterpret_cast<const uint32_t*>(u + kv_key_pair(g + 8, grp, C::RB, C::G));
                    const uint32_t s0 = __byte_perm(k0, 0, 0x1010), b0 = __byte_perm(k0, 0, 0x3232);
                    const uint32_t s1 = __byte_perm(k1, 0, 0x1010), b1 = __byte_perm(k1, 0, 0x3232);
                    uint32_t w0v[4], w1v[4];
                    constexpr int NWK = C::RB < 64 ? 2 : 4;
                    if (C::RB < 64) {
                        const uint2 x0 = lds64(u + g * 32 + t * 8), x1 = lds64(u + (g + 8) * 32 + t * 8);
                        w0v[0] = x0.x, w0v[1] = x0.y, w1v[0] = x1.x, w1v[1] = x1.y;
                    } else {
                        const uint4 x0 = lds128(u + p * 1024 + g * 64 + t * 16), x1 = lds128(u + p * 1024 + (g + 8) * 64 + t * 16);
                        w0v[0] = x0.x, w0v[1] = x0.y, w0v[2] = x0.z, w0v[3] = x0.w;
                        w1v[0] = x1.x, w1v[1] = x1.y, w1v[2] = x1.z, w1v[3] = x1.w;
                    }
#pragma unroll
                    for (int w = 0; w < NWK; ++w) {
                        if (BITS == 4) {
#pragma unroll
                            for (int hf = 0; hf < 2; ++hf) {
                                const int st = (p * NWK + w) * 2 + hf;
                                const uint32_t a0 = dequant4(w0v[w] >> (8 * hf), s0, b0), a2 = dequant4(w0v[w] >> (8 * hf + 4), s0, b0);
                                const uint32_t a1 = dequant4(w1v[w] >> (8 * hf), s1, b1), a3 = dequant4(w1v[w] >> (8 * hf + 4), s1, b1);
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) {
                                    const uint2 q = qf[(nt * C::STEPS + st) * 32 + lane];
                                    mma_bf16_16816(sc[e][nt], a0, a1, a2, a3, q.x, q.y);
                                }
                            }
                        } else {
                            const int st = p * NWK + w;
                            const uint32_t a0 = dequant8(w0v[w], s0, b0), a2 = dequant8(w0v[w] >> 8, s0, b0);
                            const uint32_t a1 = dequant8(w1v[w], s1, b1), a3 = dequant8(w1v[w] >> 8, s1, b1);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                const uint2 q = qf[(nt * C::STEPS + st) * 32 + lane];
                                mma_bf16_16816(sc[e][nt], a0, a1, a2, a3, q.x, q.y);
                            }
                        }
                    }
                }
            }
            if (!ok) break;
            // scores in units of log2, masked where a row does not see the position
            const int pos = unit_of(k) * kKvRows;
            const bool mask = pos + 2 * kKvRows > min(first_seen, s.len) || !two;
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        sc[e][nt][x] *= a.scale_log2;
                        if (mask && (pos + e * kKvRows + g + (x >> 1) * 8 >= lim[nt][x & 1] || (e == 1 && !two))) sc[e][nt][x] = -INFINITY;
                    }
            bool grew = false;
            float mu[NT][2], up_by[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float mx = fmaxf(fmaxf(sc[0][nt][x], sc[0][nt][x + 2]), fmaxf(sc[1][nt][x], sc[1][nt][x + 2]));
#pragma unroll
                    for (int of = 4; of < 32; of <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, of));
                    const float mn = fmaxf(m[nt][x], mx);
                    grew |= mn > m[nt][x];
                    mu[nt][x] = mn == -INFINITY ? 0.f : mn;
                    up_by[nt][x] = ex2(m[nt][x] - mu[nt][x]);
                    m[nt][x] = mn;
                }
            if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) l[nt][x] *= up_by[nt][x];
#pragma unroll
                    for (int j = 0; j < D / 16; ++j)
#pragma unroll
                        for (int x = 0; x < 4; ++x) o[nt][j][x] *= up_by[nt][x & 1];
                }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (e == 1 && !two) continue;
                uint32_t pb[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float p[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        p[x] = ex2(sc[e][nt][x] - mu[nt][x & 1]);
                        l[nt][x & 1] += p[x];
                    }
                    pb[nt][0] = movmatrix(bf16x2_of(p[0], p[1]));
                    pb[nt][1] = movmatrix(bf16x2_of(p[2], p[3]));
                }
                const uint8_t* u = up[e];
                constexpr int NW = C::RB / 32;  // words per lane and row
                uint32_t vw[4][NW], pr[4];
                const int key0 = pos + e * kKvRows;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int r = 2 * t + (q & 1) + (q >> 1) * 8;
                    pr[q] = *reinterpret_cast<const uint32_t*>(u + kv_value_pair(r, g * (D / 8) / 64, C::RB, C::G));
                    // a row behind the last position may hold anything; as zeros it adds nothing
                    if (key0 + r >= s.len) pr[q] = 0u;
                    const uint8_t* vb = u + kKvRows * (C::RB + 4 * C::G) + (q * 8 + t) * 16;
                    if constexpr (NW == 1) {
                        vw[q][0] = *reinterpret_cast<const uint32_t*>(vb + (g >> 2) * 64 + (g & 3) * 4);
                    } else if constexpr (NW == 2) {
                        const uint2 x = lds64(vb + (g >> 2) * 512 + ((g >> 1) & 1) * 64 + (g & 1) * 8);
                        vw[q][0] = x.x, vw[q][1] = x.y;
                    } else if constexpr (NW == 4) {
                        const uint4 x = lds128(vb + (g >> 1) * 512 + (g & 1) * 64);
                        vw[q][0] = x.x, vw[q][1] = x.y, vw[q][2] = x.z, vw[q][3] = x.w;
                    } else {  // two pieces, odd lanes take them in the other order (no bank conflict)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const uint4 x = lds128(vb + g * 512 + (c ^ (g & 1)) * 64);
                            vw[q][4 * c] = x.x, vw[q][4 * c + 1] = x.y, vw[q][4 * c + 2] = x.z, vw[q][4 * c + 3] = x.w;
                        }
                    }
                }
                const uint32_t s01 = __byte_perm(pr[0], pr[1], 0x5410), b01 = __byte_perm(pr[0], pr[1], 0x7632);
                const uint32_t s23 = __byte_perm(pr[2], pr[3], 0x5410), b23 = __byte_perm(pr[2], pr[3], 0x7632);
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    if (BITS == 4) {
#pragma unroll
                        for (int hf = 0; hf < 2; ++hf) {
                            const uint32_t x01 = __byte_perm(vw[0][w], vw[1][w], hf ? 0x7632 : 0x5410);
                            const uint32_t x23 = __byte_perm(vw[2][w], vw[3][w], hf ? 0x7632 : 0x5410);
#pragma unroll
                            for (int y = 0; y < 2; ++y) {
                                const uint32_t a0 = dequant4(x01 >> (8 * y), s01, b01), a1 = dequant4(x01 >> (8 * y + 4), s01, b01);
                                const uint32_t a2 = dequant4(x23 >> (8 * y), s23, b23), a3 = dequant4(x23 >> (8 * y + 4), s23, b23);
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt)
                                    mma_bf16_16816(o[nt][w * 4 + hf * 2 + y], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
                            }
                        }
                    } else {
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            const uint32_t s0 = 2 * y, s1 = 2 * y + 1;  // byte n of both rows to bits [0,8) and [16,24)
                            const uint32_t a0 = dequant8(__byte_perm(vw[0][w], vw[1][w], s0 | (4 + s0) << 8), s01, b01);
                            const uint32_t a1 = dequant8(__byte_perm(vw[0][w], vw[1][w], s1 | (4 + s1) << 8), s01, b01);
                            const uint32_t a2 = dequant8(__byte_perm(vw[2][w], vw[3][w], s0 | (4 + s0) << 8), s23, b23);
                            const uint32_t a3 = dequant8(__byte_perm(vw[2][w], vw[3][w], s1 | (4 + s1) << 8), s23, b23);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
                                mma_bf16_16816(o[nt][w * 2 + y], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
                        }
                    }
                }
            }
            __syncwarp();  // both slots are read by every lane before lane 0 refills them
            issue(min(mine, k + 2 + C::RING));
        }
        if (!ok) {  // a copy did not arrive (recorded): give the others in flight their time, then leave
            for (uint32_t q = done; q < done + issued; ++q) mbar_wait(&bars[q % C::RING], (q / C::RING) & 1);
            if (lane == 0) stop = 1;
        }
        done += mine;

        // join the four warps: their rows through shared memory, over the ring
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int of = 4; of < 32; of <<= 1) l[nt][x] += __shfl_xor_sync(0xffffffffu, l[nt][x], of);
        __syncthreads();
        if (stop) return;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int r = nt * 8 + 2 * t + x;
                if (g == 0) ml[warp * C::ROWS + r] = make_float2(m[nt][x], l[nt][x]);
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    // float4 i of lane g's features, placed at i 8 + (g + r & ~1) % 8: conflict-free both ways
                    int at = i;
                    if (D == 256 && BITS == 8 && (g & 1)) at = i ^ 4;  // odd lanes hold their two pieces swapped
                    merge[(warp * C::ROWS + r) * (D / 4) + at * 8 + ((g + (r & ~1)) & 7)] =
                        make_float4(o[nt][2 * i][x], o[nt][2 * i][x + 2], o[nt][2 * i + 1][x], o[nt][2 * i + 1][x + 2]);
                }
            }
        __syncthreads();
        for (int i = tid; i < nrows * (D / 4); i += kThreads) {
            const int r = i / (D / 4), f = i % (D / 4), gg = f / (D / 32), at = f % (D / 32);
            float mx = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, ml[w * C::ROWS + r].x);
            const float mr = mx == -INFINITY ? 0.f : mx;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float2 e = ml[w * C::ROWS + r];
                const float f2 = ex2(e.x - mr);
                const float4 v = merge[(w * C::ROWS + r) * (D / 4) + at * 8 + ((gg + (r & ~1)) & 7)];
                sum += f2 * e.y;
                acc.x += f2 * v.x, acc.y += f2 * v.y, acc.z += f2 * v.z, acc.w += f2 * v.w;
            }
            if (whole) {
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                const int rr = row0 + r;
                uint16_t* y = a.out + ((int64_t)(s.q0 + rr / a.group) * a.heads + h * a.group + rr % a.group) * D + f * 4;
                *reinterpret_cast<uint2*>(y) = make_uint2(bf16x2_of(acc.x * inv, acc.y * inv), bf16x2_of(acc.z * inv, acc.w * inv));
            } else {
                reinterpret_cast<float4*>(work.o)[((int64_t)slot * C::ROWS + r) * (D / 4) + f] = acc;
                if (f == 0) work.ml[slot * C::ROWS + r] = make_float2(mx, sum);
            }
        }
        fence_proxy_async_smem();  // the next range's bulk copies write where the rows were
        __syncthreads();
    }
}

// Joins a tile's partial rows.  Block (i, r): row r of the tile that share boundary i cuts, if i is the
// first boundary inside it.
template <int D>
__global__ void __launch_bounds__(256) attn_join_kernel(const __grid_constant__ AttnArgs a, int grid, int rows) {
    constexpr int F = D / 4, GROUPS = 256 / F;
    __shared__ uint32_t pre[kAttnMaxBatch + 1];
    __shared__ float wgt[2048];
    __shared__ float4 acc_s[256];
    __shared__ float red[256];
    const int tid = threadIdx.x;
    pdl_wait();
    pdl_launch_dependents();
    const StepWork work = step_work(a.part, grid, rows);
    for (int b = tid; b <= a.batch; b += 256) pre[b] = work.prefix[b];
    const uint32_t share = work.prefix[kAttnMaxBatch + 1];
    __syncthreads();
    const uint64_t w = (uint64_t)(blockIdx.x + 1) * share;
    if (w >= pre[a.batch]) return;
    int lo = 0, hi = a.batch - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (pre[mid] <= w) lo = mid; else hi = mid - 1;
    }
    const int b = lo;
    const SeqSpan s = seq_span(a, b);
    const uint32_t nu = (uint32_t)((s.len + kKvRows - 1) / kKvRows);
    const uint32_t tiles = (uint32_t)((s.n * a.group + rows - 1) / rows);
    const uint32_t ti = ((uint32_t)w - pre[b]) / nu, first = pre[b] + ti * nu;
    if (first == w || (uint64_t)blockIdx.x * share > first) return;  // no cut here, or an earlier one joins it
    const int h = (int)(ti / tiles), row = (int)(ti % tiles) * rows + (int)blockIdx.y;
    if (row >= s.n * a.group) return;
    const uint32_t c0 = first / share, n = (first + nu - 1) / share - c0 + 1;
    auto slot_of = [&](uint32_t i) { return 2 * (c0 + i) + ((uint64_t)(c0 + i) * share >= first ? 0 : 1); };
    float mx = -INFINITY;
    for (uint32_t i = tid; i < n; i += 256) mx = fmaxf(mx, work.ml[slot_of(i) * rows + blockIdx.y].x);
    red[tid] = mx;
    __syncthreads();
    for (int o = 128; o; o >>= 1) {
        if (tid < o) red[tid] = fmaxf(red[tid], red[tid + o]);
        __syncthreads();
    }
    mx = red[0] == -INFINITY ? 0.f : red[0];
    __syncthreads();
    float sum = 0.f;
    for (uint32_t i = tid; i < n; i += 256) {
        const float2 e = work.ml[slot_of(i) * rows + blockIdx.y];
        const float f = ex2(e.x - mx);
        wgt[i] = f;
        sum += f * e.y;
    }
    red[tid] = sum;
    __syncthreads();
    for (int o = 128; o; o >>= 1) {
        if (tid < o) red[tid] += red[tid + o];
        __syncthreads();
    }
    sum = red[0];
    const int f = tid % F, grp = tid / F;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (uint32_t i = grp; i < n; i += GROUPS) {
        const float4 v = reinterpret_cast<const float4*>(work.o)[((int64_t)slot_of(i) * rows + blockIdx.y) * F + f];
        const float g = wgt[i];
        acc.x += g * v.x, acc.y += g * v.y, acc.z += g * v.z, acc.w += g * v.w;
    }
    acc_s[tid] = acc;
    __syncthreads();
    if (grp) return;
    for (int i = 1; i < GROUPS; ++i) {
        const float4 v = acc_s[i * F + f];
        acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    uint16_t* y = a.out + ((int64_t)(s.q0 + row / a.group) * a.heads + h * a.group + row % a.group) * D + f * 4;
    *reinterpret_cast<uint2*>(y) = make_uint2(bf16x2_of(acc.x * inv, acc.y * inv), bf16x2_of(acc.z * inv, acc.w * inv));
}

template <typename... P, typename... A>
cudaError_t launch_attn(void (*kernel)(P...), dim3 grid, int threads, uint32_t smem, bool pdl, cudaStream_t stream, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

constexpr int kStepMaxCtas = 5;  // per SM, the most of any StepCfg

template <int D, int BITS, int NT>
cudaError_t run_step(const AttnArgs& a, cudaStream_t stream) {
    using C = StepCfg<D, BITS, NT>;
    cudaError_t e = cudaFuncSetAttribute(attn_step_kernel<D, BITS, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM);
    if (e != cudaSuccess) return e;
    // no more CTAs than the longest lengths the table can hold would occupy
    const int64_t tiles = (int64_t)a.pool.kv_heads * (a.tokens * a.group / C::ROWS + a.batch);
    const int64_t most = tiles * a.table_width * a.pool.page_units;
    const int grid = (int)std::max<int64_t>(1, std::min<int64_t>((int64_t)device_num_sms() * C::CTAS, (most + kMinShare - 1) / kMinShare));
    e = launch_attn(attn_step_kernel<D, BITS, NT>, dim3(grid), kThreads, C::SMEM, a.pdl, stream, a);
    if (e != cudaSuccess || grid == 1) return e;
    return launch_attn(attn_join_kernel<D>, dim3(grid - 1, C::ROWS), 256, 0, a.pdl, stream, a, grid, (int)C::ROWS);
}

template <int D, int BITS>
cudaError_t run_rows(const AttnArgs& a, cudaStream_t stream) {
    return (int64_t)a.max_q * a.group <= 8 ? run_step<D, BITS, 1>(a, stream) : run_step<D, BITS, 2>(a, stream);
}

}  // namespace

size_t attn_workspace_bytes(int64_t tokens, int heads, int kv_heads, int dim, int batch) {
    return kStepHead + (size_t)2 * device_num_sms() * kStepMaxCtas * 16 * (dim * 4 + 8);
}

bool attention_applies(const AttnArgs& a) {
    const int64_t tiles = (int64_t)a.pool.kv_heads * (a.tokens * a.group / 8 + a.batch);
    return (double)tiles * a.table_width * a.pool.page_units < 4.0e9;
}

cudaError_t launch_paged_attention(const AttnArgs& a, cudaStream_t stream) {
    const bool b4 = a.pool.bits == 4;
    if (a.pool.dim == 64) return b4 ? run_rows<64, 4>(a, stream) : run_rows<64, 8>(a, stream);
    if (a.pool.dim == 128) return b4 ? run_rows<128, 4>(a, stream) : run_rows<128, 8>(a, stream);
    return b4 ? run_rows<256, 4>(a, stream) : run_rows<256, 8>(a, stream);
}

int attn_device_error(bool clear) { return tu_device_error(clear); }

}  // namespace marlin
