// attn_chunk.cu — attention of many query rows over the paged, quantized cache (prompts, chunks of
// prompts, long drafts) on the 5th-generation tensor cores.
//
// A tile is 128 rows of one (sequence, kv head): its (token, head of the group) pairs in order, so grouped
// heads share every dequantized key and value.  Per step of 128 cached positions:
//   S[128 x 128] = Q K^T        tcgen05.mma kind::f16, Q and K in shared memory, S in TMEM (two or three buffers)
//   P = 2^(c S - M + e)         one thread per row, written back over S as f16
//   O[128 x dim] += P V         P from TMEM, V in shared memory (features contiguous: an MN-major operand)
// Keys and values are dequantized to f16 (11 bits, one rounding of scale * code + bias) rather than bf16:
// the largest bias of a unit of 16 positions gives a power of two that puts it in range, 2^eK for its keys,
// folded into the softmax factor c of its columns, 2^e for its values, folded into their exponent; M is the
// running maximum of (c S + e), so a unit with small values never loses its weights' bits.  Each query row
// is scaled by its own power of two.  M moves only when a row outgrows it by 2^8, which keeps the rescaling
// of O rare.
//
// Bound: tensor pipe (dim 256: 2048 cycles a step), the exponentials (128 x 128 at 16 a cycle and SM: 1024)
// or the issue slots of dequantizing (about 2 instructions per cached value and tile).
// Warps: 0-7 softmax and output (two threads per row, 64 columns each, who agree on M through shared
// memory), the next 4 or 8 dequantize, each its own units, codes prefetched to registers one step ahead
// straight from the pages, and one issues the MMAs.  Items (tile, range of steps) are laid out by a planning kernel from
// the lengths on the device: no more steps per item than an SM's fair share, longest tiles first, taken by
// persistent CTAs from a counter; a tile of several items is joined from binary32 partial rows in item order.
#include <algorithm>

#include "attn_common.cuh"
#include "q4_host.cuh"

namespace marlin {
namespace {

constexpr int kRows = 128;       // rows of a tile (M)
constexpr int kKeys = 128;       // positions of a step
constexpr int kSoft = 8;         // softmax warps
constexpr int kWarpDeq = 8;      // first dequantizing warp
constexpr int kItemCost = 2;     // fixed cost of an item (queries, pipeline fill, output), in steps
constexpr uint32_t kTmemCols = 512;
constexpr float kLazy = 8.f;     // log2 of how far a row may outgrow its maximum before O is rescaled

struct Item {
    int b, row0;   // sequence, first row of the tile
    int k0, k1;    // steps
    int slot;      // partial rows, -1: the whole tile
    int pad[3];
};
struct Cut {       // a tile of several items
    int b, row0, slot, n;
};
// Workspace: counters, items (per kv head the same ones), cuts, then per slot kRows (M, l) and [kRows][dim].
struct ChunkWork {
    int* head;     // [0] next item, [1] items, [2] cuts
    Item* items;
    Cut* cuts;
    float2* ml;
    float* o;
};
inline int64_t tiles_most(int64_t tokens, int group, int batch) { return tokens * group / kRows + batch; }
// Items beyond one per tile come from cut tiles; a cut tile of s steps gives at most 2 s / limit items and
// limit >= total / SMs, so over all heads cut tiles give at most 2 SMs items (plus one per head for rounding).
__host__ __device__ inline int64_t slots_most(int sms, int kv_heads) { return 2 * (int64_t)sms / kv_heads + 2; }

inline ChunkWork chunk_work(float* part, int64_t tiles, int sms, int kv_heads) {
    uint8_t* p = reinterpret_cast<uint8_t*>(part);
    auto take = [&](size_t n) {
        uint8_t* q = p;
        p += (n + 255) / 256 * 256;
        return q;
    };
    const int64_t slots = slots_most(sms, kv_heads);
    ChunkWork w;
    w.head = reinterpret_cast<int*>(take(256));
    w.items = reinterpret_cast<Item*>(take((tiles + slots) * sizeof(Item)));
    w.cuts = reinterpret_cast<Cut*>(take(slots * sizeof(Cut)));
    w.ml = reinterpret_cast<float2*>(take((size_t)slots * kv_heads * kRows * sizeof(float2)));
    w.o = reinterpret_cast<float*>(p);
    return w;
}

// Steps of the tile whose first row is row0: up to the last position any of its rows sees.
__device__ __forceinline__ int tile_steps(const SeqSpan& s, int row0, int group) {
    const int last = min(s.n * group, row0 + kRows) - 1;
    const int seen = min(s.len, s.len - s.n + last / group + 1);
    return seen <= 0 ? 0 : (seen + kKeys - 1) / kKeys;
}

// Exclusive prefix sum over the 1024 threads of the block; returns the total through `all`.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* tmp, uint32_t& all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) tmp[warp] = x;
    __syncthreads();
    uint32_t w = tmp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += y;
    }
    all = __shfl_sync(0xffffffffu, w, 31);
    const uint32_t before = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
    return x - v + (warp ? before : 0u);
}

// One block lays out the items.
__global__ void __launch_bounds__(1024) attn_plan_kernel(const __grid_constant__ AttnArgs a, ChunkWork w, int64_t tiles_cap, int sms) {
    __shared__ uint32_t tmp[32];
    __shared__ int first_tile[kAttnMaxBatch + 1];
    __shared__ SeqSpan span[kAttnMaxBatch];
    const int tid = threadIdx.x;
    pdl_wait();
    pdl_launch_dependents();
    SeqSpan s{0, 0, 0};
    if (tid < a.batch) {
        s = seq_span(a, tid);
        span[tid] = s;
    }
    uint32_t ntiles;
    const uint32_t at = block_scan((uint32_t)((s.n * a.group + kRows - 1) / kRows), tmp, ntiles);
    if (tid < a.batch) first_tile[tid] = (int)at;
    if (tid == 0) first_tile[a.batch] = (int)ntiles;
    __syncthreads();
    // starts that overlap could ask for more tiles than the tokens fill
    const int tiles = (int)min((int64_t)ntiles, tiles_cap);
    if (tid == 0 && tiles < (int64_t)ntiles) record_device_error(kDevErrBadIndex);
    auto tile_of = [&](int i, int& b, int& row0) {
        int lo = 0, hi = a.batch - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (first_tile[mid] <= i) lo = mid; else hi = mid - 1;
        }
        b = lo;
        row0 = (i - first_tile[lo]) * kRows;
        return tile_steps(span[lo], row0, a.group);
    };
    uint32_t total = 0;
    for (int i0 = 0; i0 < tiles; i0 += 1024) {
        int b, row0;
        uint32_t all;
        block_scan(i0 + tid < tiles ? (uint32_t)(tile_of(i0 + tid, b, row0) + kItemCost) : 0u, tmp, all);
        total += all;
    }
    const uint32_t limit = max(4u, (uint32_t)(((uint64_t)total * a.pool.kv_heads + sms - 1) / sms));
    uint32_t items = 0, slots = 0, cuts = 0;
    for (int i0 = 0; i0 < tiles; i0 += 1024) {
        const int i = i0 + tid;
        int b = 0, row0 = 0, steps = 0;
        uint32_t n = 0;
        if (i < tiles) {  // later rows of a sequence see more: last tiles first
            steps = tile_of(tiles - 1 - i, b, row0);
            n = max(1u, (steps + limit - 1) / limit);
        }
        uint32_t ni, ns, nc;
        const uint32_t ai = items + block_scan(n, tmp, ni), as = slots + block_scan(n > 1 ? n : 0u, tmp, ns);
        const uint32_t ac = cuts + block_scan(n > 1 ? 1u : 0u, tmp, nc);
        for (uint32_t j = 0; j < n; ++j) {
            Item it{};
            it.b = b;
            it.row0 = row0;
            it.k0 = (int)((uint64_t)steps * j / n);
            it.k1 = (int)((uint64_t)steps * (j + 1) / n);
            it.slot = n > 1 ? (int)(as + j) : -1;
            w.items[ai + j] = it;
        }
        if (n > 1) w.cuts[ac] = Cut{b, row0, (int)as, (int)n};
        items += ni, slots += ns, cuts += nc;
    }
    if (tid == 0) {
        w.head[0] = 0;
        w.head[1] = (int)items;
        w.head[2] = (int)cuts;
    }
}

template <int D, int BITS>
struct ChunkCfg {
    static constexpr int RB = kv_row_bytes(D, BITS), G = D / 64, UB = kv_unit_bytes(D, BITS);
    static constexpr int NB = D == 256 ? 1 : 2;           // dequantized K and V buffers
    static constexpr int SB = D == 256 ? 2 : 3;           // S buffers in TMEM (128 columns each, O behind them)
    static constexpr int DW = 8;                          // dequantizing warps
    static constexpr int UPW = 8 / DW;                    // units of a step per dequantizing warp
    static constexpr int KC = RB / 32;                    // 16-byte pieces per lane and unit
    // 8-bit codes of many features would take 64 registers for a step: V follows K through the same ones
    static constexpr bool ONE = D == 256 && BITS == 8;
    // Warpgroups: two softmax, one or two dequantizing, and one whose first warp issues the MMAs.  The issuer
    // hands its registers to the others (the launch's total: 512 x 128 or 640 x 96).
    static constexpr int WARP_MMA = kWarpDeq + DW, THREADS = (WARP_MMA + 4) * 32;
    static constexpr int REGS_SOFT = D == 256 ? 112 : 128, REGS_DEQ = D == 256 ? 112 : 96, REGS_MMA = 24;
    static constexpr int REGS_ALL = (kSoft * REGS_SOFT + DW * REGS_DEQ + 4 * REGS_MMA) * 32;
    static_assert(REGS_ALL <= THREADS * 96);
    static constexpr uint32_t QB = kRows * D * 2, KB = kKeys * D * 2;
    static constexpr uint32_t OFF_K = QB, OFF_V = OFF_K + NB * KB, OFF_T = OFF_V + NB * KB;
    static constexpr uint32_t TAB = 2 * 8 * 2 * G * 16 * 4;  // f16 (scale, bias): [2 steps][unit][K, V][group][row]
    static constexpr bool KEEP = D <= 128;                // a softmax thread keeps its 64 scores in registers
    static constexpr uint32_t OFF_E = OFF_T + TAB;        // exponents [4 steps][unit]: 2^eK, e, 2^-e
    static constexpr uint32_t OFF_X = OFF_E + 4 * 8 * 16; // [2 steps][half][row]: maxima of the two halves of a row
    static constexpr uint32_t OFF_SR = OFF_X + 2 * 2 * kRows * 4;
    static constexpr uint32_t OFF_BAR = OFF_SR + kRows * 4;
    static constexpr uint32_t SMEM = 1024 + OFF_BAR + 256;
};

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
          "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
          "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// Shared-memory descriptor of an MN-major operand, 128-byte swizzle: 64 features of one position per
// 128-byte line, 8-position atoms of 1024 B (stride), 64-feature panels `panel` bytes apart (leading).
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(const void* smem_ptr, uint32_t panel) {
    const uint64_t addr = smem_u32(smem_ptr);
    return ((addr & 0x3FFFFull) >> 4) | ((uint64_t)(panel >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
constexpr uint32_t kIdescBMn = 1u << 16;  // B is MN-major

// the two warps of a TMEM lane quarter
__device__ __forceinline__ void pair_barrier(int quarter) { asm volatile("bar.sync %0, 64;" ::"r"(quarter + 1) : "memory"); }

__device__ __forceinline__ uint32_t f16x2_fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
__device__ __forceinline__ uint32_t f16x2_mul(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

// A 16-byte piece of one row's codes -> f16 (scale * code + bias), 16-byte lines of eight features each, at
// lines c0, c0 + 1, ... of the row at `row` (128-byte swizzle by the row).  With 4 bits a line's features
// stand in the order 0, 4, 1, 5, 2, 6, 3, 7 (the order they unpack in; queries and outputs follow it).
template <int BITS>
__device__ __forceinline__ void dequant_piece(const uint4& x, uint32_t pair, uint8_t* row, uint32_t c0, uint32_t sw) {
    const uint32_t s2 = __byte_perm(pair, 0, 0x1010), b2 = __byte_perm(pair, 0, 0x3232);
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    if (BITS == 4) {
        const uint32_t s16 = f16x2_mul(s2, 0x2C002C00u);  // scale / 16
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t o[4];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const uint32_t v = y ? w[i] >> 8 : w[i];
                o[2 * y] = f16x2_fma(f16x2_add(lop3_and_or(v, 0x000F000Fu, kF16Magic), 0xE400E400u), s2, b2);
                o[2 * y + 1] = f16x2_fma(f16x2_add(lop3_and_or(v, 0x00F000F0u, kF16Magic), 0xE400E400u), s16, b2);
            }
            *reinterpret_cast<uint4*>(row + (((c0 + i) ^ sw) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t o[4];
#pragma unroll
            for (int y = 0; y < 4; ++y)
                o[y] = f16x2_fma(f16x2_add(__byte_perm(w[2 * i + (y >> 1)], kF16MagicBytes, y & 1 ? 0x4342 : 0x4140), 0xE400E400u), s2, b2);
            *reinterpret_cast<uint4*>(row + (((c0 + i) ^ sw) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
}

// two binary32 at once
__device__ __forceinline__ uint64_t f32x2(float lo, float hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
    return d;
}
__device__ __forceinline__ void f32x2_split(uint64_t v, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t f32x2_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t f32x2_add(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

template <int REGS>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS)); }
template <int REGS>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS)); }

template <int D, int BITS>
__global__ void __launch_bounds__(ChunkCfg<D, BITS>::THREADS, 1)
    attn_chunk_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ ChunkWork work) {
    using C = ChunkCfg<D, BITS>;
    constexpr int G = C::G, NB = C::NB, SB = C::SB, KC = C::KC, DW = C::DW, UPW = C::UPW, kWarpMma = C::WARP_MMA;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = align_smem_1024(smem_raw);
    uint8_t* sq = smem;
    uint8_t* sk = smem + C::OFF_K;
    uint8_t* sv = smem + C::OFF_V;
    uint32_t* tab = reinterpret_cast<uint32_t*>(smem + C::OFF_T);
    float4* expo = reinterpret_cast<float4*>(smem + C::OFF_E);
    float* xch = reinterpret_cast<float*>(smem + C::OFF_X);
    float* qsr = reinterpret_cast<float*>(smem + C::OFF_SR);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
    uint64_t* kfull = bars;            // [NB] dequantizing warps
    uint64_t* kfree = kfull + NB;      // [NB] MMA commit
    uint64_t* vfull = kfree + NB;      // [NB]
    uint64_t* vfree = vfull + NB;      // [NB] MMA commit: P V of the step done
    uint64_t* sfull = vfree + NB;      // [SB] MMA commit
    uint64_t* pfull = sfull + SB;      // [SB] softmax warps
    uint64_t* efull = pfull + SB;      // [4] dequantizing warps: the step's exponents (they run up to 3 steps ahead)
    uint64_t* pdone = efull + 4;       // [SB] MMA commit: P V of the step (and of all before it) done
    uint64_t* fin = pdone + SB;        // [1]
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_s, item_s;
    volatile int* abort = &abort_s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (warp == kWarpMma) {
        tmem_alloc(&tmem_slot, kTmemCols);
        tmem_relinquish();
    }
    if (tid == 0) {
        abort_s = 0;
        for (int i = 0; i < NB; ++i) {
            mbar_init(&kfull[i], DW);
            mbar_init(&kfree[i], 1);
            mbar_init(&vfull[i], DW);
            mbar_init(&vfree[i], 1);
        }
        for (int i = 0; i < SB; ++i) {
            mbar_init(&sfull[i], 1);
            mbar_init(&pdone[i], 1);
            mbar_init(&pfull[i], kSoft);
        }
        for (int i = 0; i < 4; ++i) mbar_init(&efull[i], DW);
        mbar_init(fin, 1);
        fence_mbar_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot, tmem_o = tmem + SB * kKeys;
    pdl_wait();
    pdl_launch_dependents();
    const int total = work.head[1] * a.pool.kv_heads;

    // Every warp meets the others three times an item: number known, queries in place, item done.
    auto sync_all = [] { asm volatile("bar.sync 0, %0;" ::"n"(C::THREADS) : "memory"); };
    // Queries, by all but the last warpgroup: D / 8 lanes per row, scaled by a power of two to a maximum in [2^10, 2^11)
    auto load_queries = [&](const Item& it, const SeqSpan& s, int h, int nrows) {
        constexpr int LPR = D / 8, RPW = 32 / LPR;
        for (int r0 = warp * RPW; r0 < kRows; r0 += (kSoft + DW) * RPW) {
            const int r = r0 + lane / LPR, c = lane % LPR;
            uint4 x = make_uint4(0u, 0u, 0u, 0u);
            if (r < nrows) {
                const int rr = it.row0 + r;
                x = *reinterpret_cast<const uint4*>(a.q + (int64_t)(s.q0 + rr / a.group) * a.q_ts +
                                                    (int64_t)(h * a.group + rr % a.group) * a.q_hs + c * 8);
            }
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
            uint32_t big = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) big = max(big, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
#pragma unroll
            for (int o = 1; o < LPR; o <<= 1) big = max(big, __shfl_xor_sync(0xffffffffu, big, o));
            const int e = max((int)(big >> 7) - 127, -100) - 10;
            const float f = pow2i(max(-e, -126));
            float v[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = __uint_as_float(w[i] << 16) * f;
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u) * f;
            }
            uint4 y;
            if (BITS == 4)
                y = make_uint4(f16x2_of(v[0], v[4]), f16x2_of(v[1], v[5]), f16x2_of(v[2], v[6]), f16x2_of(v[3], v[7]));
            else
                y = make_uint4(f16x2_of(v[0], v[1]), f16x2_of(v[2], v[3]), f16x2_of(v[4], v[5]), f16x2_of(v[6], v[7]));
            *reinterpret_cast<uint4*>(sq + (c >> 3) * (kRows * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = y;
            if (c == 0) qsr[r] = a.scale_log2 * pow2i(min(e, 127));
        }
        fence_proxy_async_smem();
    };
    uint32_t base = 0;  // steps of the CTA's earlier items (barrier phases run on)

    if (warp < kWarpDeq) {
        regs_up<C::REGS_SOFT>();
        for (;;) {
            if (tid == 0) item_s = *abort ? total : atomicAdd(&work.head[0], 1);
            sync_all();
            const int id = item_s;
            if (id >= total) break;
            const Item it = work.items[id / a.pool.kv_heads];
            const int h = id % a.pool.kv_heads, n = it.k1 - it.k0;
            const SeqSpan s = seq_span(a, it.b);
            const int nrows = min(kRows, s.n * a.group - it.row0);
            load_queries(it, s, h, nrows);
            sync_all();
            const int quarter = warp & 3, half = warp >> 2;
            const uint32_t lane_base = (uint32_t)(32 * quarter) << 16;
            const int r = quarter * 32 + lane, rr = it.row0 + r;
            const float sr = qsr[r];
            const int lim = r < nrows ? min(s.len, s.len - s.n + rr / a.group + 1) : 0;
            const int low = min(s.len, s.len - s.n + (it.row0 + quarter * 32) / a.group + 1);  // the warp's first row sees least
            const bool short_tile = quarter * 32 + 32 > nrows;
            const uint32_t oc = tmem_o + lane_base + half * (D / 2);  // this thread's columns of O
            float m = -INFINITY, l = 0.f;
            bool ok = true;
            for (int j = 0; j < n; ++j) {
                const uint32_t gj = base + j;
                const int pos = (it.k0 + j) * kKeys + half * 64;
                // on an abort the pair still meets at its barrier, once a step
                ok = ok && warp_wait<true>(&efull[gj & 3], (gj / 4) & 1, abort) && warp_wait<true>(&sfull[gj % SB], (gj / SB) & 1, abort);
                if (!ok) {
                    pair_barrier(quarter);
                    continue;
                }
                tc_fence_after();
                const float4* ex = expo + (gj & 3) * 8 + half * 4;
                const uint32_t ts = tmem + lane_base + (gj % SB) * kKeys + half * 64;
                const bool mask = pos + 64 > low || short_tile;
                // scores of columns 32 q .. 32 q + 31, -inf where the row does not see the position
                uint32_t x[C::KEEP ? 64 : 32];
                auto fetch = [&](int q, uint32_t (&v)[32]) {
                    tmem_ld32(ts + q * 32, v);
                    tmem_wait_ld();
                    if (mask) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (pos + q * 32 + i >= lim) v[i] = 0xff800000u;
                    }
                };
                float xm = -INFINITY;
                if constexpr (C::KEEP) {
                    tmem_ld32(ts, reinterpret_cast<uint32_t(&)[32]>(x[0]));
                    tmem_ld32(ts + 32, reinterpret_cast<uint32_t(&)[32]>(x[32]));
                    tmem_wait_ld();
                    if (mask) {
#pragma unroll
                        for (int i = 0; i < 64; ++i)
                            if (pos + i >= lim) x[i] = 0xff800000u;
                    }
                }
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    if constexpr (!C::KEEP) fetch(q, reinterpret_cast<uint32_t(&)[32]>(x));
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const uint32_t* z = x + (C::KEEP ? q * 32 : 0) + y * 16;
                        float m0 = __uint_as_float(z[0]), m1 = __uint_as_float(z[1]);
#pragma unroll
                        for (int i = 2; i < 16; i += 4) {
                            m0 = fmaxf(fmaxf(m0, __uint_as_float(z[i])), __uint_as_float(z[i + 1]));
                            if (i + 2 < 16) m1 = fmaxf(fmaxf(m1, __uint_as_float(z[i + 2])), __uint_as_float(z[i + 3]));
                        }
                        m0 = fmaxf(m0, m1);
                        const float4 e = ex[q * 2 + y];
                        if (m0 > -INFINITY) xm = fmaxf(xm, fmaf(m0, sr * e.x, e.y));
                    }
                }
                float* xc = xch + (gj & 1) * (2 * kRows);
                xc[half * kRows + r] = xm;
                pair_barrier(quarter);
                xm = fmaxf(xm, xc[(half ^ 1) * kRows + r]);
                const bool grow = xm > m + kLazy || (m == -INFINITY && xm > -INFINITY);
                if (__any_sync(0xffffffffu, grow)) {
                    const float by = grow ? ex2(m - xm) : 1.f;  // 0 from -inf
                    if (j > 0) {
                        ok = warp_wait<true>(&pdone[(gj - 1) % SB], ((gj - 1) / SB) & 1, abort);
                        tc_fence_after();
#pragma unroll 1
                        for (int q = 0; q < D / 32; ++q) {
                            uint32_t z[16];
                            tmem_ld16(oc + q * 16, z);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; ++i) z[i] = __float_as_uint(__uint_as_float(z[i]) * by);
                            tmem_st16(oc + q * 16, z);
                        }
                    }
                    l *= by;
                    if (grow) m = xm;
                }
                const float mm = m == -INFINITY ? 0.f : m;
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    if constexpr (!C::KEEP) fetch(q, reinterpret_cast<uint32_t(&)[32]>(x));
                    uint32_t p[16];
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const uint32_t* z = x + (C::KEEP ? q * 32 : 0) + y * 16;
                        const float4 e = ex[q * 2 + y];
                        const uint64_t c = f32x2(sr * e.x, sr * e.x), off = f32x2(e.y - mm, e.y - mm);
                        uint64_t sum = 0;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            float p0, p1;
                            f32x2_split(f32x2_fma(f32x2(__uint_as_float(z[2 * i]), __uint_as_float(z[2 * i + 1])), c, off), p0, p1);
                            p0 = ex2(p0);
                            p1 = ex2(p1);
                            sum = f32x2_add(sum, f32x2(p0, p1));
                            p[8 * y + i] = f16x2_of(p0, p1);
                        }
                        float s0, s1;
                        f32x2_split(sum, s0, s1);
                        l = fmaf(s0 + s1, e.z, l);
                    }
                    tmem_st16(ts + q * 16, p);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&pfull[gj % SB]);
            }
            // output: half of this thread's row
            if (n > 0 && ok) ok = warp_wait<true>(&pdone[(base + n - 1) % SB], ((base + n - 1) / SB) & 1, abort);
            tc_fence_after();
            float* xc = xch + ((base + n) & 1) * (2 * kRows);
            xc[half * kRows + r] = l;
            pair_barrier(quarter);
            if (ok) {
                l += xc[(half ^ 1) * kRows + r];
                const bool whole = it.slot < 0;
                const int slot = it.slot * a.pool.kv_heads + h;
                const float inv = l == 0.f ? 0.f : 1.f / l;
                uint16_t* y = a.out + ((int64_t)(s.q0 + rr / a.group) * a.heads + h * a.group + rr % a.group) * D + half * (D / 2);
                float* po = work.o + ((int64_t)slot * kRows + r) * D + half * (D / 2);
                if (!whole && r < nrows && half == 0) work.ml[(int64_t)slot * kRows + r] = make_float2(m, l);
#pragma unroll 1
                for (int q = 0; q < D / 64; ++q) {
                    uint32_t x[32];
                    if (n > 0) {
                        tmem_ld32(oc + q * 32, x);
                        tmem_wait_ld();
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) x[i] = 0u;
                    }
                    if (r < nrows) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float v[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i)  // back to the features' own order
                                v[i] = __uint_as_float(x[8 * e + (BITS == 4 ? (i & 3) * 2 + (i >> 2) : i)]);
                            if (whole) {
                                *reinterpret_cast<uint4*>(y + q * 32 + e * 8) =
                                    make_uint4(bf16x2_of(v[0] * inv, v[1] * inv), bf16x2_of(v[2] * inv, v[3] * inv),
                                               bf16x2_of(v[4] * inv, v[5] * inv), bf16x2_of(v[6] * inv, v[7] * inv));
                            } else {
                                float4* z = reinterpret_cast<float4*>(po + q * 32 + e * 8);
                                z[0] = make_float4(v[0], v[1], v[2], v[3]);
                                z[1] = make_float4(v[4], v[5], v[6], v[7]);
                            }
                        }
                    }
                    __syncwarp();
                }
            }
            tc_fence_before();
            base += n;
            sync_all();  // queries, TMEM and the item's number are free for the next item
            tc_fence_after();
        }
    } else if (warp < kWarpMma) {
        regs_up<C::REGS_DEQ>();
        for (;;) {
            sync_all();
            const int id = item_s;
            if (id >= total) break;
            const Item it = work.items[id / a.pool.kv_heads];
            const int h = id % a.pool.kv_heads, n = it.k1 - it.k0;
            const SeqSpan s = seq_span(a, it.b);
            const int nrows = min(kRows, s.n * a.group - it.row0);

            // dequantizing warps: the codes of the first step on their way before anything else
            const int dw = warp - kWarpDeq, pu = a.pool.page_units;
            uint4 kr[UPW][KC], vr[C::ONE ? 1 : UPW][KC];
            uint32_t pr[UPW][G];
            const uint8_t* ua[UPW];          // the units of the step whose keys are loaded last
            const uint8_t* uv[UPW];          // those of the step whose values are loaded next
            int pi[UPW], ri[UPW], pg[UPW];   // page and unit in the page one step further, and its table entry
            int last_page = 0;
            auto fetch_pages = [&]() {       // entries behind the last position repeat the last page (masked later)
#pragma unroll
                for (int u = 0; u < UPW; ++u) pg[u] = a.table[(int64_t)it.b * a.table_stride + min(pi[u], last_page)];
            };
            auto next_units = [&]() {        // looks at the entries only now: their load is a step old
#pragma unroll
                for (int u = 0; u < UPW; ++u) {
                    if (pg[u] < 0 || pg[u] >= a.pool.pages) {
                        record_device_error(kDevErrBadIndex);
                        pg[u] = 0;
                    }
                    ua[u] = a.pool.data + (((int64_t)pg[u] * a.pool.kv_heads + h) * pu + ri[u]) * (int64_t)C::UB;
                    pi[u] += 8 / pu;
                    ri[u] += 8 % pu;
                    if (ri[u] >= pu) {
                        ri[u] -= pu;
                        ++pi[u];
                    }
                }
            };
            auto load_pr = [&]() {  // lanes 0-15: the keys' rows, 16-31: the values'
#pragma unroll
                for (int u = 0; u < UPW; ++u) {
                    const uint8_t* p = ua[u] + (lane < 16 ? kv_key_pair(lane, 0, C::RB, G) : kv_value_pair(lane - 16, 0, C::RB, G));
                    if constexpr (G == 4) {
                        const uint4 x = __ldg(reinterpret_cast<const uint4*>(p));
                        pr[u][0] = x.x, pr[u][1] = x.y, pr[u][2] = x.z, pr[u][3] = x.w;
                    } else if constexpr (G == 2) {
                        const uint2 x = __ldg(reinterpret_cast<const uint2*>(p));
                        pr[u][0] = x.x, pr[u][1] = x.y;
                    } else {
                        pr[u][0] = __ldg(reinterpret_cast<const uint32_t*>(p));
                    }
                }
            };
            // A warp's 512 bytes: keys 8 rows of one 64-byte panel (or all 16 of a 32-byte row), values two
            // pieces of all 16 rows; eight neighbouring lanes hold eight rows (no bank conflict when they store).
            const int krow = C::RB >= 64 ? lane & 7 : (lane & 7) + 8 * (lane >> 4);
            const int vrow = (lane & 3) * 2 + ((lane >> 2) & 1) + 8 * (lane >> 4);
            auto load_k = [&]() {
#pragma unroll
                for (int u = 0; u < UPW; ++u)
#pragma unroll
                    for (int i = 0; i < KC; ++i)
                        kr[u][i] = __ldg(reinterpret_cast<const uint4*>(
                            ua[u] + (C::RB >= 64 ? (i >> 1) * 1024 + (i & 1) * 512 + krow * 64 + (lane >> 3) * 16 : krow * 32 + ((lane >> 3) & 1) * 16)));
            };
            auto load_v = [&](uint4 (&r)[UPW][KC]) {
#pragma unroll
                for (int u = 0; u < UPW; ++u)
#pragma unroll
                    for (int i = 0; i < KC; ++i)
                        r[u][i] = __ldg(reinterpret_cast<const uint4*>(uv[u] + kKvRows * (C::RB + 4 * G) + i * 512 + (lane >> 4) * 256 +
                                                                       ((lane >> 2) & 1) * 128 + ((lane >> 3) & 1) * 64 + (lane & 3) * 16));
            };
            if (n > 0) {
                last_page = ((s.len + kKvRows - 1) / kKvRows - 1) / pu;
#pragma unroll
                for (int u = 0; u < UPW; ++u) {
                    const int unit = it.k0 * 8 + dw * UPW + u;
                    pi[u] = unit / pu;
                    ri[u] = unit % pu;
                }
                fetch_pages();
                next_units();
                if (n > 1) fetch_pages();
                load_pr();
                load_k();
#pragma unroll
                for (int u = 0; u < UPW; ++u) uv[u] = ua[u];
                if constexpr (!C::ONE) load_v(vr);
            }
            load_queries(it, s, h, nrows);
            sync_all();
            // Keys run one step ahead of values: K of step j + 1 while P V of step j - 1 runs, V of step j while
            // Q K^T of step j + 1 does, so that one buffer of each (dim 256) keeps the tensor pipe fed.
            bool ok = true;  // warp-uniform
            auto keys = [&](int j) {
                const uint32_t gj = base + j, st = gj % NB, use = gj / NB;
                // exponents and f16 (scale, bias) of this warp's units, of keys and values
#pragma unroll
                for (int u = 0; u < UPW; ++u) {
                    const int unit = dw * UPW + u, row = lane & 15, isv = lane >> 4;
                    uint32_t big = 0;
#pragma unroll
                    for (int i = 0; i < G; ++i) {
                        if ((it.k0 + j) * kKeys + unit * kKvRows + row >= s.len) pr[u][i] = 0u;  // behind the last position: zeros
                        const uint32_t sc = pr[u][i] & 0x7fffu, bi = (pr[u][i] >> 16) & 0x7fffu;
                        // |value| <= max(|bias|, 16 or 256 |scale|) up to a factor of two
                        big = max(big, max(bi, sc ? sc + (BITS << 7) : 0u));
                    }
                    // 2^-e puts the largest into [2^10, 2^12)
                    const int ek = max((int)(__reduce_max_sync(0xffffffffu, isv ? 0u : big) >> 7) - 137, -100);
                    const int ev = max((int)(__reduce_max_sync(0xffffffffu, isv ? big : 0u) >> 7) - 137, -100);
                    const float f = pow2i(max(isv ? -ev : -ek, -126));
                    uint32_t* t = tab + (((gj & 1) * 8 + unit) * 2 + isv) * (G * 16) + row;
#pragma unroll
                    for (int i = 0; i < G; ++i)
                        t[i * 16] = f16x2_of(__uint_as_float(pr[u][i] << 16) * f, __uint_as_float(pr[u][i] & 0xffff0000u) * f);
                    if (lane == 0) expo[(gj & 3) * 8 + unit] = make_float4(pow2i(min(ek, 127)), (float)ev, pow2i(max(-ev, -126)), 0.f);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&efull[gj & 3]);
                ok = ok && (use == 0 || warp_wait<true>(&kfree[st], (use - 1) & 1, abort));
                if (ok) {
                    uint8_t* kb = sk + st * C::KB;
#pragma unroll
                    for (int u = 0; u < UPW; ++u)
#pragma unroll
                        for (int i = 0; i < KC; ++i) {
                            const int unit = dw * UPW + u, row = C::RB >= 64 ? (i & 1) * 8 + krow : krow;
                            const int dim = (C::RB >= 64 ? (i >> 1) * 64 + (lane >> 3) * 16 : ((lane >> 3) & 1) * 16) * 8 / BITS;
                            dequant_piece<BITS>(kr[u][i], tab[(((gj & 1) * 8 + unit) * 2 * G + (dim >> 6)) * 16 + row],
                                                kb + (dim >> 6) * (kKeys * 128) + (unit * 16 + row) * 128, (dim & 63) >> 3, row & 7);
                        }
                    fence_proxy_async_smem();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&kfull[st]);
            };
            auto load_keys = [&](int j) {  // of step j, and the table entries of the one after
                next_units();
                if (j + 1 < n) fetch_pages();
                load_pr();
                load_k();
            };
            if (n > 0) keys(0);
            if (n > 1) load_keys(1);
            for (int j = 0; j < n && ok; ++j) {
                const uint32_t gj = base + j, st = gj % NB, use = gj / NB;
                if (j + 1 < n) keys(j + 1);
                if constexpr (C::ONE) {
                    load_v(kr);
                } else {
#pragma unroll
                    for (int u = 0; u < UPW; ++u) uv[u] = ua[u];
                    if (j + 2 < n) load_keys(j + 2);
                }
                ok = ok && (use == 0 || warp_wait<true>(&vfree[st], (use - 1) & 1, abort));
                if (ok) {
                    uint8_t* vb = sv + st * C::KB;
#pragma unroll
                    for (int u = 0; u < UPW; ++u)
#pragma unroll
                        for (int i = 0; i < KC; ++i) {
                            const int unit = dw * UPW + u, dim = (i * 2 + ((lane >> 3) & 1)) * 128 / BITS;
                            const uint4& x = C::ONE ? kr[u][i] : vr[C::ONE ? 0 : u][i];
                            dequant_piece<BITS>(x, tab[((((gj & 1) * 8 + unit) * 2 + 1) * G + (dim >> 6)) * 16 + vrow],
                                                vb + (dim >> 6) * (kKeys * 128) + (unit * 16 + vrow) * 128, (dim & 63) >> 3, vrow & 7);
                        }
                    fence_proxy_async_smem();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&vfull[st]);
                if constexpr (C::ONE) {
#pragma unroll
                    for (int u = 0; u < UPW; ++u) uv[u] = ua[u];
                    if (j + 2 < n) load_keys(j + 2);
                } else {
                    if (j + 1 < n) load_v(vr);
                }
            }
            base += n;
            sync_all();
        }
    } else {
        regs_down<C::REGS_MMA>();
        for (;;) {
            sync_all();
            const int id = item_s;
            if (id >= total) break;
            const Item it = work.items[id / a.pool.kv_heads];
            const int n = it.k1 - it.k0;
            sync_all();
            tc_fence_after();
            if (warp == kWarpMma && lane == 0 && n > 0) {
                const uint32_t idesc_s = umma_idesc_f16(kRows, kKeys), idesc_o = umma_idesc_f16(kRows, D) | kIdescBMn;
                const uint64_t qd = umma_desc_sw128(sq), kd0 = umma_desc_sw128(sk), vd0 = umma_desc_mn_sw128(sv, kKeys * 128);
                auto qk = [&](int j) {
                    const uint32_t gj = base + j, st = gj % NB;
                    if (!thread_wait<true>(&kfull[st], (gj / NB) & 1, abort)) return false;
                    // S of step j goes where P of step j - SB stands: that product has to be done
                    if (gj >= SB && !thread_wait<true>(&pdone[gj % SB], (gj / SB - 1) & 1, abort)) return false;
                    tc_fence_after();
                    const uint64_t kd = kd0 + (uint64_t)((st * C::KB) >> 4);
#pragma unroll 1  // short loops: unrolled, the issuer waits for its instructions (16 products 3100 cycles)
                    for (int p = 0; p < D / 64; ++p)
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint64_t off = (uint64_t)(p * (kRows * 128 >> 4) + k * 2);
                            umma_smem_a(tmem + (gj % SB) * kKeys, qd + off, kd + off, idesc_s, p > 0 || k > 0);
                        }
                    umma_commit(&kfree[st]);
                    umma_commit(&sfull[gj % SB]);
                    return true;
                };
                bool ok = qk(0);
                for (int j = 0; j < n && ok; ++j) {
                    if (j + 1 < n && !(ok = qk(j + 1))) break;
                    const uint32_t gj = base + j, st = gj % NB;
                    ok = thread_wait<true>(&vfull[st], (gj / NB) & 1, abort) && thread_wait<true>(&pfull[gj % SB], (gj / SB) & 1, abort);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t vd = vd0 + (uint64_t)((st * C::KB) >> 4);
#pragma unroll 1
                    for (int p = 0; p < 2; ++p)  // P: 64 positions in 32 columns at the start of each half of S
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            umma_tmem_a(tmem_o, tmem + (gj % SB) * kKeys + p * 64 + k * 8, vd + (uint64_t)((p * 4 + k) * (16 * 128 >> 4)),
                                        idesc_o, j > 0 || p > 0 || k > 0);
                    umma_commit(&vfree[st]);
                    umma_commit(&pdone[gj % SB]);
                }
            }
            __syncwarp();
            base += n;
            sync_all();
        }
    }
    if (warp == kWarpMma) {
        if (lane == 0) {
            umma_commit(fin);  // every MMA issued above completes before TMEM is released
            drain_wait(fin, 0);
        }
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

// Joins the rows of cut tiles: block (cut, kv head, 16-row part), a warp per row.
template <int D>
__global__ void __launch_bounds__(256) attn_chunk_join_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ ChunkWork work) {
    pdl_wait();
    pdl_launch_dependents();
    if ((int)blockIdx.x >= work.head[2]) return;
    const Cut c = work.cuts[blockIdx.x];
    const int h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const SeqSpan s = seq_span(a, c.b);
    for (int i = 0; i < 2; ++i) {
        const int r = blockIdx.z * 16 + warp * 2 + i, rr = c.row0 + r;
        if (rr >= s.n * a.group) continue;
        auto at = [&](int k) { return ((int64_t)(c.slot + k) * a.pool.kv_heads + h) * kRows + r; };
        float mx = -INFINITY;
        for (int k = lane; k < c.n; k += 32) mx = fmaxf(mx, work.ml[at(k)].x);
#pragma unroll
        for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        if (mx == -INFINITY) mx = 0.f;
        float sum = 0.f, acc[D / 32] = {};
#pragma unroll 4
        for (int k = 0; k < c.n; ++k) {
            const float2 e = work.ml[at(k)];
            const float f = ex2(e.x - mx);
            sum += f * e.y;
            const float2* o = reinterpret_cast<const float2*>(work.o + at(k) * D);
#pragma unroll
            for (int q = 0; q < D / 64; ++q) {
                const float2 v = o[q * 32 + lane];
                acc[2 * q] += f * v.x;
                acc[2 * q + 1] += f * v.y;
            }
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        uint16_t* y = a.out + ((int64_t)(s.q0 + rr / a.group) * a.heads + h * a.group + rr % a.group) * D;
#pragma unroll
        for (int q = 0; q < D / 64; ++q)
            reinterpret_cast<uint32_t*>(y)[q * 32 + lane] = bf16x2_of(acc[2 * q] * inv, acc[2 * q + 1] * inv);
    }
}

template <typename... P, typename... A>
cudaError_t launch_chunk(void (*kernel)(P...), dim3 grid, int threads, uint32_t smem, bool pdl, cudaStream_t stream, A... args) {
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

template <int D, int BITS>
cudaError_t run_chunk(const AttnArgs& a, cudaStream_t stream) {
    using C = ChunkCfg<D, BITS>;
    cudaError_t e = cudaFuncSetAttribute(attn_chunk_kernel<D, BITS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM);
    if (e != cudaSuccess) return e;
    // the warpgroups' register shares have to fit what the block is launched with, or their increase waits for good
    static const int regs = [] {
        cudaFuncAttributes f{};
        return cudaFuncGetAttributes(&f, attn_chunk_kernel<D, BITS>) == cudaSuccess ? f.numRegs : 0;
    }();
    if (regs * C::THREADS < C::REGS_ALL) return cudaErrorInvalidConfiguration;
    const int sms = device_num_sms();
    const int64_t tiles = tiles_most(a.tokens, a.group, a.batch);
    const ChunkWork w = chunk_work(a.part, tiles, sms, a.pool.kv_heads);
    e = launch_chunk(attn_plan_kernel, dim3(1), 1024, 0, a.pdl, stream, a, w, tiles, sms);
    if (e != cudaSuccess) return e;
    e = launch_chunk(attn_chunk_kernel<D, BITS>, dim3(sms), C::THREADS, C::SMEM, a.pdl, stream, a, w);
    if (e != cudaSuccess) return e;
    const int64_t cuts = std::min(tiles, slots_most(sms, a.pool.kv_heads) / 2);
    return launch_chunk(attn_chunk_join_kernel<D>, dim3((unsigned)cuts, a.pool.kv_heads, kRows / 16), 256, 0, a.pdl, stream, a, w);
}

}  // namespace

bool chunk_fits(const AttnArgs& a) {
    // items of all heads, and the plan's sum of steps, in 31 bits
    const double tiles = (double)tiles_most(a.tokens, a.group, a.batch) + slots_most(device_num_sms(), a.pool.kv_heads);
    const double steps = (double)a.table_width * a.pool.page_units * kKvRows / kKeys + 1 + kItemCost;
    return tiles * a.pool.kv_heads < 2.0e9 && tiles * steps < 2.0e9;
}

size_t chunk_workspace_bytes(int64_t tokens, int heads, int kv_heads, int dim, int batch) {
    const int sms = device_num_sms();
    const ChunkWork w = chunk_work(nullptr, tiles_most(tokens, heads / kv_heads, batch), sms, kv_heads);
    return reinterpret_cast<size_t>(w.o) + (size_t)slots_most(sms, kv_heads) * kv_heads * kRows * dim * 4;
}

cudaError_t launch_attn_chunk(const AttnArgs& a, cudaStream_t stream) {
    const bool b4 = a.pool.bits == 4;
    if (a.pool.dim == 64) return b4 ? run_chunk<64, 4>(a, stream) : run_chunk<64, 8>(a, stream);
    if (a.pool.dim == 128) return b4 ? run_chunk<128, 4>(a, stream) : run_chunk<128, 8>(a, stream);
    return b4 ? run_chunk<256, 4>(a, stream) : run_chunk<256, 8>(a, stream);
}

int chunk_device_error(bool clear) { return tu_device_error(clear); }

}  // namespace marlin
