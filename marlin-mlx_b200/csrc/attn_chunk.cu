// attn_chunk.cu — attention of many query rows over the paged, quantized cache (prompts, chunks of
// prompts, long drafts) on the 5th-generation tensor cores.
//
// A tile is 128 rows of one (sequence, kv head): its (token, head of the group) pairs in order, so grouped
// heads share every dequantized key and value.  Per step of 128 cached positions:
//   S[128 x 128] = Q K^T        tcgen05.mma kind::f16, Q and K in shared memory, S in TMEM (two or three buffers)
//   P = 2^(c S - M + e)         one thread per row, written back over S as f16
//   O[128 x dim] += P V         P from TMEM, V in shared memory (features contiguous: an MN-major operand)
// Keys and values are dequantized to f16 (11 bits, one rounding of scale * code + bias) rather than bf16:
// the tile's largest bias gives a power of two that puts them in range, 2^eK for a step's keys, folded into
// the softmax factor c, 2^e for its values, folded into the exponent; M is the running maximum of
// (c S + e), so a step with small values never loses its weights' bits.  Each query row is scaled by its own
// power of two.  M moves only when a row outgrows it by 2^8, which keeps the rescaling of O rare.
//
// Bound: tensor pipe (dim 256: 2048 cycles a step), the exponentials (128 x 128 at 16 a cycle and SM: 1024)
// or the issue slots of dequantizing (about 2 instructions per cached value and tile).
// Warps: 0-3 softmax and output, 4 issues the MMAs, 5-12 dequantize (codes prefetched to registers one step
// ahead, straight from the pages).  Items (tile, range of steps) are laid out by a planning kernel from the
// lengths on the device: no more steps per item than an SM's fair share, longest tiles first, taken by
// persistent CTAs from a counter; a tile of several items is joined from binary32 partial rows in item order.
#include <algorithm>

#include "attn_common.cuh"
#include "q4_host.cuh"

namespace marlin {
namespace {

constexpr int kRows = 128;       // rows of a tile (M)
constexpr int kKeys = 128;       // positions of a step
constexpr int kSoft = 4;         // softmax warps
constexpr int kWarpMma = 4;
constexpr int kDeq = 8;          // dequantizing warps, from warp 5
constexpr int kThreads = (kSoft + 1 + kDeq) * 32;
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
    static constexpr int KC = RB / 32;                    // 16-byte pieces per dequantizing thread and step
    static constexpr uint32_t QB = kRows * D * 2, KB = kKeys * D * 2;
    static constexpr uint32_t OFF_K = QB, OFF_V = OFF_K + NB * KB, OFF_T = OFF_V + NB * KB;
    static constexpr uint32_t TAB = 2 * G * kKeys * 4;    // f16 (scale, bias) of a step: [K, V][group][position]
    static constexpr uint32_t OFF_SR = OFF_T + 2 * TAB;
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

__device__ __forceinline__ void deq_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(kDeq * 32) : "memory"); }

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

template <int D, int BITS>
__global__ void __launch_bounds__(kThreads, 1) attn_chunk_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ ChunkWork work) {
    using C = ChunkCfg<D, BITS>;
    constexpr int G = C::G, NB = C::NB, SB = C::SB, KC = C::KC;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = align_smem_1024(smem_raw);
    uint8_t* sq = smem;
    uint8_t* sk = smem + C::OFF_K;
    uint8_t* sv = smem + C::OFF_V;
    uint32_t* tab = reinterpret_cast<uint32_t*>(smem + C::OFF_T);
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
    uint64_t* fin = pdone + SB;         // [1]
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_s, item_s;
    __shared__ uint32_t emax[4][2];
    __shared__ float expo[4][2];       // 2^eK, eV of a step
    volatile int* abort = &abort_s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (warp == kWarpMma) {
        tmem_alloc(&tmem_slot, kTmemCols);
        tmem_relinquish();
    }
    if (tid == 0) {
        abort_s = 0;
        for (int i = 0; i < NB; ++i) {
            mbar_init(&kfull[i], kDeq);
            mbar_init(&kfree[i], 1);
            mbar_init(&vfull[i], kDeq);
            mbar_init(&vfree[i], 1);
        }
        for (int i = 0; i < SB; ++i) {
            mbar_init(&sfull[i], 1);
            mbar_init(&pdone[i], 1);
            mbar_init(&pfull[i], kSoft);
        }
        for (int i = 0; i < 4; ++i) mbar_init(&efull[i], kDeq);
        mbar_init(fin, 1);
        fence_mbar_init();
    }
    if (tid < 8) emax[tid >> 1][tid & 1] = 0u;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot, tmem_o = tmem + SB * kKeys;
    pdl_wait();
    pdl_launch_dependents();
    const int total = work.head[1] * a.pool.kv_heads;

    uint32_t base = 0;  // steps of the CTA's earlier items (barrier phases run on)
    for (;;) {
        if (tid == 0) item_s = *abort ? total : atomicAdd(&work.head[0], 1);
        __syncthreads();
        const int id = item_s;
        if (id >= total) break;
        const Item it = work.items[id / a.pool.kv_heads];
        const int h = id % a.pool.kv_heads;
        const SeqSpan s = seq_span(a, it.b);
        const int n = it.k1 - it.k0;
        const int nrows = min(kRows, s.n * a.group - it.row0);
        const int nu = (s.len + kKvRows - 1) / kKvRows;

        // dequantizing warps: the codes of the first step on their way before anything else
        const int dw = warp - 5;
        uint4 kr[KC], vr[KC];
        uint32_t pr[G];
        const uint8_t* ua = nullptr;  // unit (lane & 7) of the step whose loads come next
        int page = 0;                 // its table entry, read a step earlier
        auto fetch_page = [&](int j) {
            const int u = min((it.k0 + j) * 8 + (lane & 7), nu - 1);
            page = table_page(a, it.b, u / a.pool.page_units);
        };
        auto unit_at = [&](int j) {
            const int u = min((it.k0 + j) * 8 + (lane & 7), nu - 1);
            ua = a.pool.data + (((int64_t)page * a.pool.kv_heads + h) * a.pool.page_units + u % a.pool.page_units) * (int64_t)C::UB;
        };
        auto unit_ptr = [&](int u) { return reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(ua), u)); };
        auto load_pr = [&]() {  // this thread's position (tid mod 128) of K (first 128 threads) or V
            const int key = (dw & 3) * 32 + lane;
            const uint64_t lo = reinterpret_cast<uint64_t>(ua);
            const uint8_t* p0 = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, lo, key >> 4));
            const uint8_t* p = p0 + (dw < 4 ? kv_key_pair(key & 15, 0, C::RB, G) : kv_value_pair(key & 15, 0, C::RB, G));
            if constexpr (G == 4) {
                const uint4 x = __ldg(reinterpret_cast<const uint4*>(p));
                pr[0] = x.x, pr[1] = x.y, pr[2] = x.z, pr[3] = x.w;
            } else if constexpr (G == 2) {
                const uint2 x = __ldg(reinterpret_cast<const uint2*>(p));
                pr[0] = x.x, pr[1] = x.y;
            } else {
                pr[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
            }
        };
        auto load_k = [&]() {
#pragma unroll
            for (int i = 0; i < KC; ++i) {
                const int blk = dw + 8 * i;
                if (C::RB >= 64) {  // 8 rows x one 64-byte panel
                    const int rowblk = blk & 15, panel = blk >> 4;
                    const uint8_t* u = unit_ptr(rowblk >> 1);
                    kr[i] = __ldg(reinterpret_cast<const uint4*>(u + panel * 1024 + ((rowblk & 1) * 8 + (lane & 7)) * 64 + (lane >> 3) * 16));
                } else {            // 16 rows x 32 bytes
                    const uint8_t* u = unit_ptr(blk);
                    kr[i] = __ldg(reinterpret_cast<const uint4*>(u + ((lane & 7) + 8 * (lane >> 4)) * 32 + ((lane >> 3) & 1) * 16));
                }
            }
        };
        auto load_v = [&]() {
#pragma unroll
            for (int i = 0; i < KC; ++i) {  // 512 bytes: two pieces of each of a unit's 16 rows
                const int blk = dw + 8 * i, u8 = blk & 7, pair = blk >> 3;
                const uint8_t* u = unit_ptr(u8);
                vr[i] = __ldg(reinterpret_cast<const uint4*>(u + kKvRows * (C::RB + 4 * G) + pair * 512 + (lane >> 4) * 256 +
                                                             ((lane >> 2) & 1) * 128 + ((lane >> 3) & 1) * 64 + (lane & 3) * 16));
            }
        };
        // exponents and f16 (scale, bias) of step j from pr, in two parts around a barrier
        auto prep_max = [&](int j) {
            const int key = (dw & 3) * 32 + lane;
            uint32_t big = 0;
#pragma unroll
            for (int i = 0; i < G; ++i) {
                if ((it.k0 + j) * kKeys + key >= s.len) pr[i] = 0u;  // behind the last position: zeros
                const uint32_t sc = pr[i] & 0x7fffu, bi = (pr[i] >> 16) & 0x7fffu;
                // |value| <= max(|bias|, 16 or 256 |scale|) up to a factor of two
                big = max(big, max(bi, sc ? sc + (BITS << 7) : 0u));
            }
            big = __reduce_max_sync(0xffffffffu, big);
            if (lane == 0) atomicMax(&emax[(base + j) & 3][dw < 4 ? 0 : 1], big);
        };
        auto prep_table = [&](int j) {
            const int key = (dw & 3) * 32 + lane;
            const uint32_t at = (base + j) & 3;
            // 2^-e puts the largest into [2^10, 2^12)
            const int e = max((int)(emax[at][dw < 4 ? 0 : 1] >> 7) - 127 - 10, -100);
            const float f = pow2i(max(-e, -126));
            uint32_t* t = tab + (((base + j) & 1) * 2 + (dw < 4 ? 0 : 1)) * (G * kKeys) + key;
#pragma unroll
            for (int i = 0; i < G; ++i)
                t[i * kKeys] = f16x2_of(__uint_as_float(pr[i] << 16) * f, __uint_as_float(pr[i] & 0xffff0000u) * f);
            if ((dw & 3) == 0 && lane == 0) expo[at][dw < 4 ? 0 : 1] = dw < 4 ? pow2i(min(e, 127)) : (float)e;
        };
        if (warp > kWarpMma && n > 0) {
            fetch_page(0);
            unit_at(0);
            load_pr();
            load_k();
            load_v();
            if (n > 1) fetch_page(1);
        }

        // queries: D / 8 lanes per row, scaled by a power of two to a maximum in [2^10, 2^11)
        if (warp != kWarpMma) {
            constexpr int LPR = D / 8, RPW = 32 / LPR;
            const int wi = warp < kWarpMma ? warp : warp - 1;
            for (int r0 = wi * RPW; r0 < kRows; r0 += (kSoft + kDeq) * RPW) {
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
        }
        __syncthreads();

        if (warp == kWarpMma) {
            if (lane == 0 && n > 0) {
                const uint32_t idesc_s = umma_idesc_f16(kRows, kKeys), idesc_o = umma_idesc_f16(kRows, D) | kIdescBMn;
                const uint64_t qd = umma_desc_sw128(sq), kd0 = umma_desc_sw128(sk), vd0 = umma_desc_mn_sw128(sv, kKeys * 128);
                auto qk = [&](int j) {
                    const uint32_t gj = base + j, st = gj % NB;
                    if (!thread_wait<true>(&kfull[st], (gj / NB) & 1, abort)) return false;
                    // S of step j goes where P of step j - SB stands: that product has to be done
                    if (gj >= SB && !thread_wait<true>(&pdone[gj % SB], (gj / SB - 1) & 1, abort)) return false;
                    tc_fence_after();
                    const uint64_t kd = kd0 + (uint64_t)((st * C::KB) >> 4);
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const uint64_t off = (uint64_t)(((k >> 2) * (kRows * 128) + (k & 3) * 32) >> 4);
                        umma_smem_a(tmem + (gj % SB) * kKeys, qd + off, kd + off, idesc_s, k > 0);
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
#pragma unroll
                    for (int k = 0; k < kKeys / 16; ++k)
                        umma_tmem_a(tmem_o, tmem + (gj % SB) * kKeys + k * 8, vd + (uint64_t)((k * 16 * 128) >> 4), idesc_o, j > 0 || k > 0);
                    umma_commit(&vfree[st]);
                    umma_commit(&pdone[gj % SB]);
                }
            }
        } else if (warp > kWarpMma) {
            bool ok = true;
            if (n > 0) {
                prep_max(0);
                deq_barrier();
                prep_table(0);
                if (tid == 5 * 32) emax[(base + 1) & 3][0] = emax[(base + 1) & 3][1] = 0u;
                __syncwarp();
                if (lane == 0) mbar_arrive(&efull[base & 3]);
                deq_barrier();
            }
            for (int j = 0; j < n; ++j) {
                const uint32_t gj = base + j, st = gj % NB, use = gj / NB;
                const uint32_t* t = tab + (gj & 1) * (2 * G * kKeys);
                const bool more = j + 1 < n;
                // ok stays warp-uniform; on an abort the warps still meet at every barrier
                ok = ok && (use == 0 || warp_wait<true>(&kfree[st], (use - 1) & 1, abort));
                uint8_t* kb = sk + st * C::KB;
                if (ok) {
#pragma unroll
                    for (int i = 0; i < KC; ++i) {
                        const int blk = dw + 8 * i;
                        int key, dim;  // dim: first feature of the piece
                        if (C::RB >= 64) {
                            key = (blk & 15) * 8 + (lane & 7);
                            dim = ((blk >> 4) * 64 + (lane >> 3) * 16) * 8 / BITS;
                        } else {
                            key = blk * 16 + (lane & 7) + 8 * (lane >> 4);
                            dim = ((lane >> 3) & 1) * 32;
                        }
                        dequant_piece<BITS>(kr[i], t[(dim >> 6) * kKeys + key], kb + (dim >> 6) * (kKeys * 128) + key * 128, (dim & 63) >> 3, key & 7);
                    }
                    fence_proxy_async_smem();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&kfull[st]);
                if (more) {
                    unit_at(j + 1);
                    load_pr();
                    load_k();
                    if (j + 2 < n) fetch_page(j + 2);
                }
                ok = ok && (use == 0 || warp_wait<true>(&vfree[st], (use - 1) & 1, abort));
                uint8_t* vb = sv + st * C::KB;
                if (ok) {
#pragma unroll
                    for (int i = 0; i < KC; ++i) {
                        const int blk = dw + 8 * i, c = (blk >> 3) * 2 + ((lane >> 3) & 1);
                        const int key = (blk & 7) * 16 + (lane & 3) * 2 + ((lane >> 2) & 1) + 8 * (lane >> 4);
                        const int dim = c * 128 / BITS;
                        dequant_piece<BITS>(vr[i], t[(G + (dim >> 6)) * kKeys + key], vb + (dim >> 6) * (kKeys * 128) + key * 128, (dim & 63) >> 3, key & 7);
                    }
                    fence_proxy_async_smem();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&vfull[st]);
                if (more) {
                    load_v();
                    prep_max(j + 1);
                    deq_barrier();
                    prep_table(j + 1);
                    if (tid == 5 * 32) emax[(gj + 2) & 3][0] = emax[(gj + 2) & 3][1] = 0u;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&efull[(gj + 1) & 3]);
                    deq_barrier();
                }
            }
        } else {
            const uint32_t lane_base = (uint32_t)(32 * warp) << 16;
            const int r = warp * 32 + lane, rr = it.row0 + r;
            const float sr = qsr[r];
            const int lim = r < nrows ? min(s.len, s.len - s.n + rr / a.group + 1) : 0;
            const int low = min(s.len, s.len - s.n + (it.row0 + warp * 32) / a.group + 1);  // the warp's first row sees least
            float m = -INFINITY, l = 0.f;
            bool ok = true;
            for (int j = 0; j < n; ++j) {
                const uint32_t gj = base + j;
                const int pos = (it.k0 + j) * kKeys;
                ok = warp_wait<true>(&efull[gj & 3], (gj / 4) & 1, abort) && warp_wait<true>(&sfull[gj % SB], (gj / SB) & 1, abort);
                if (!ok) break;
                tc_fence_after();
                const float c = sr * expo[gj & 3][0], ev = expo[gj & 3][1];
                const uint32_t ts = tmem + lane_base + (gj % SB) * kKeys;
                const bool mask = pos + kKeys > low || r >= nrows;
                float mx = -INFINITY;
                uint32_t x[32];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    tmem_ld32(ts + q * 32, x);
                    tmem_wait_ld();
                    if (__any_sync(0xffffffffu, mask)) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) mx = fmaxf(mx, pos + q * 32 + i < lim ? __uint_as_float(x[i]) : -INFINITY);
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) mx = fmaxf(mx, __uint_as_float(x[i]));
                    }
                }
                const float xm = mx == -INFINITY ? -INFINITY : fmaf(mx, c, ev);
                const bool grow = xm > m + kLazy || (m == -INFINITY && xm > -INFINITY);
                if (__any_sync(0xffffffffu, grow)) {
                    const float by = grow ? ex2(m - xm) : 1.f;  // 0 from -inf
                    if (j > 0) {
                        if (!(ok = warp_wait<true>(&pdone[(gj - 1) % SB], ((gj - 1) / SB) & 1, abort))) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int q = 0; q < D / 32; ++q) {
                            tmem_ld32(tmem_o + lane_base + q * 32, x);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * by);
                            tmem_st32(tmem_o + lane_base + q * 32, x);
                        }
                    }
                    l *= by;
                    if (grow) m = xm;
                }
                const float off = m == -INFINITY ? 0.f : ev - m;
                float sum = 0.f;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    tmem_ld32(ts + q * 32, x);
                    tmem_wait_ld();
                    uint32_t p[16];
                    if (__any_sync(0xffffffffu, mask)) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (pos + q * 32 + i >= lim) x[i] = 0xff800000u;  // -inf
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float p0 = ex2(fmaf(__uint_as_float(x[2 * i]), c, off)), p1 = ex2(fmaf(__uint_as_float(x[2 * i + 1]), c, off));
                        sum += p0 + p1;
                        p[i] = f16x2_of(p0, p1);
                    }
                    tmem_st16(ts + q * 16, p);
                }
                l = fmaf(sum, ex2(-ev), l);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&pfull[gj % SB]);
            }
            // output: this thread's row
            if (n > 0 && ok) ok = warp_wait<true>(&pdone[(base + n - 1) % SB], ((base + n - 1) / SB) & 1, abort);
            tc_fence_after();
            if (ok) {
                const bool whole = it.slot < 0;
                const int slot = it.slot * a.pool.kv_heads + h;
                const float inv = l == 0.f ? 0.f : 1.f / l;
                uint16_t* y = a.out + ((int64_t)(s.q0 + rr / a.group) * a.heads + h * a.group + rr % a.group) * D;
                float* po = work.o + ((int64_t)slot * kRows + r) * D;
                if (!whole && r < nrows) work.ml[(int64_t)slot * kRows + r] = make_float2(m, l);
#pragma unroll 1
                for (int q = 0; q < D / 32; ++q) {
                    uint32_t x[32];
                    if (n > 0) {
                        tmem_ld32(tmem_o + lane_base + q * 32, x);
                        tmem_wait_ld();
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) x[i] = 0u;
                    }
                    if (r < nrows)
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
                    __syncwarp();
                }
            }
            tc_fence_before();
        }
        base += n;
        __syncthreads();  // queries, TMEM and the item's number are free for the next item
        tc_fence_after();
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
    const int sms = device_num_sms();
    const int64_t tiles = tiles_most(a.tokens, a.group, a.batch);
    const ChunkWork w = chunk_work(a.part, tiles, sms, a.pool.kv_heads);
    e = launch_chunk(attn_plan_kernel, dim3(1), 1024, 0, a.pdl, stream, a, w, tiles, sms);
    if (e != cudaSuccess) return e;
    e = launch_chunk(attn_chunk_kernel<D, BITS>, dim3(sms), kThreads, C::SMEM, a.pdl, stream, a, w);
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
