// Attention of several new tokens per sequence on B200 tensor cores (tcgen05), with TMA and tensor
// memory; kvb_chunk.cuh has the definition. fp16 or int8 pages, or packed fp16 keys and values; fp32 or
// fp16 queries; head dims 64 and 128.
//
// A query tile is 128 rows, (token, query head of one KV head's group), so that one load of a key tile
// serves the whole group; a unit is two query tiles and 128-key tiles of their keys. Per key tile
//     S[128 rows x 128 keys] = Q K^T      (Q, K in shared memory, K-major)
//     P = exp2(f S - m), l += row sums
//     O[128 rows x D] += P V              (P in tensor memory, V in shared memory, MN-major)
// with the running reference m of a row raised only when a tile's probabilities sum to more than 2^14 (then O
// and l are scaled in place), so O stays in tensor memory and the common tile needs no maximum; a row without a
// reference yet is raised by its first finite score. One
// persistent CTA per SM, 16 warps:
//   0-3, 4-7   softmax of query tiles 0 and 1, one thread per row (tensor-memory lane).
//   8          unit scheduler, and TMA producer of the key tiles and the query tiles.
//   9          TMA producer of the value tiles (with small pages one warp's issue of 16 boxes a tile was slower
//              than the memory).
//   10, 11     one elected thread each issues the score products and the value products. (A lane chosen by
//              its number instead of elect.sync took 85 cycles a product, longer than the product, and one
//              thread for both kinds was the bottleneck: with its share of waits and commits it took 2000
//              cycles a key tile and query tile, twice the products' time.) With split operands (QF32) a
//              tile's scores and probabilities share their columns, and warp 10 issues both kinds in order.
//   12-15      fp16 values: non-finite elements of tiles that some row does not see in full are set to 0
//              (0 x inf would not be 0) and, where a row does see them, added at the end. int8: tiles
//              converted to fp16 (exact); the scales are applied to the scores and to the probabilities.
// fp32 queries (QF32) keep fp32-level results: q and p are split as fp16(x) + fp16(x - fp16(x)) (about 22
// bits; q prescaled per row by a power of two) and both products run on both halves.
//
// What bounds it: at head dim 128 the four products of a pair of query tiles take 2048 cycles a key tile and
// the exponentials as many, and a pair takes about 3700: neither pipe is full (55 %), since a tile's
// probabilities are handed over once and its value product starts behind the last of them. A prompt of 8192
// tokens (32 heads over 8, 0.55 TFLOP that count): 447-459 us in a burst and 520 in a loop of seconds, whose
// clock the 1 kW power cap lowers (1230 and 1060 TFLOP/s; library products 1653 and 1375); 2048 tokens on a
// 32 k context: 904 and 1075 us (1180 and 990 TFLOP/s); 512 fp32 queries on 32 k of int8 pages: 630 and 619
// us, 870 TFLOP/s of the products with split operands (fp16 queries: 475 us; fp16 pages: 243 us. Converting
// the tiles and their scales are more code than the instruction cache holds beside the rest). Few tokens on
// long contexts are bound by a tile's chain of scores, exponentials and value product, with one of the two
// softmax groups idle in units of one query tile (8 ragged chunks, 311 MB: 76 us, 4.1 TB/s, on pages of 16 and
// of 128 tokens alike) and, at the smallest, by the start, first loads and the join (4 x 3-8 tokens on 4 k, 57
// MB: 28 us).
#include <cuda.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "kvb_chunk.cuh"
#include "kvb_tc.cuh"

namespace {

using namespace kvb_dev;

constexpr int CU_ROWS = 128;            // query rows of a tile, keys of a tile
constexpr int CU_SUB = CU_ROWS * 128;   // bytes of [128 rows][128 B], one 128-byte-swizzled slice
constexpr int CU_RING = 2;              // units in flight between the roles
// One pair of probabilities in so many is computed on the FMA pipe instead of the exponential unit. At head dim
// 64 the products are half as long and the exponentials are what a tile takes (prompt of 8192 tokens: 464 us
// without, 439 with one in 8, 446 in 4, 513 in 2); at 128 the products are, and it costs (444 -> 439, but 2048
// tokens on 32 k 948 -> 983).
template <int D>
constexpr int CU_POLY_OF = D == 64 ? 8 : 0;
constexpr int CU_CLEAN = 8;             // value tiles on their way to the cleaning warps: at most their stages are
enum { SRC_F16 = 0, SRC_I8 = 1, SRC_PACKED = 2 };
// The tensor cores add into O with truncation, an error of up to 2^-23 of O per product of 16 keys and in
// one direction. So O is added into an fp32 sum in the workspace (rounded to nearest) and started anew
// every so many key tiles: often for fp32 results, rarely for fp16 ones. (512 fp32 queries on 32 k int8:
// relative error 3.5e-5 and 3.5e-6 for the plain fp32 form; folded every 8, 12, 16 tiles 3.6e-6, 4.5e-6,
// 5.6e-6 and 647, 609, 605 us: 12 trades 1e-6 of error for 6 % of the time.)
constexpr int CU_FOLD_F32 = KVB_CHUNK_FOLD_F32, CU_FOLD_F16 = KVB_CHUNK_FOLD_F16;
// A row's highest score at its reference's last move has probability 2^CU_SHIFT, so that small ones stay normal
// in fp16.
constexpr float CU_SHIFT = 5.f;
constexpr float CU_MOST = 16384.f;  // a key tile's probabilities of a row may sum to this before the reference moves

// The work of a call is a line: sequence by sequence, KV head by KV head, unit by unit, each unit as long as
// its cost (keys, and an overhead), cut into equal parts, one per CTA. So every CTA ends at about the same
// time whatever the lengths, and a call with few units splits their keys. A unit that a cut goes through
// (at a key tile) is computed in pieces, which a second small kernel joins. (Whole units handed out longest
// first, their keys split evenly only where units were fewer than SMs: 250 us instead of 112 for 8 chunks of
// 1-256 tokens on contexts of 512-30000, and 948 instead of 923 for 2048 tokens on 32 k.) Costs are in quarter
// keys: a unit with one query tile counts three quarters.
constexpr long long CU_COST_UNIT = 4 * 480;       // a unit's overhead: its queries' load, first maximum, output
constexpr long long CU_COST_LEAST = 4 * 512;      // work that is worth a CTA
constexpr int CU_SNAP = 2;                        // no cut nearer than this to a unit's first or last key tile

// The first k units of a sequence (of one KV head) on that line.
__device__ __forceinline__ long long cost_upto(const ChunkParams& p, const ChunkSeq& s, long long k) {
    if (s.bad) return k * CU_COST_UNIT;
    if (s.n <= p.tile_tokens) return k * (CU_COST_UNIT + 3ll * (s.ctx + s.n));
    return k * (CU_COST_UNIT + 4ll * s.ctx) + 2ll * p.unit_tokens * k * (k + 1);
}
__device__ __forceinline__ int seq_units(const ChunkParams& p, const ChunkSeq& s) {
    return s.bad ? 1 : (s.n + p.unit_tokens - 1) / p.unit_tokens;
}

// Where the cut at x of a unit of cost w falls among its nt key tiles.
__device__ __forceinline__ int cut_tile(long long x, long long w, int nt) {
    if (x <= 0) return 0;
    if (x >= w) return nt;
    const int k = int(x * nt / w);
    return k < CU_SNAP ? 0 : k > nt - CU_SNAP ? nt : k;
}

template <int SRC, bool QF32, int D>
struct CCfg {
    static constexpr int NSUB = D / 64;
    static constexpr int ITEM = NSUB * CU_SUB;              // one K or V tile in fp16
    static constexpr int QTILE = NSUB * CU_SUB * (QF32 ? 2 : 1);
    static constexpr int RAW = CU_ROWS * D;                 // one int8 tile
    static constexpr int BUDGET = 227 * 1024 - 1024 - 2048;  // alignment, small arrays
    // Stages of K and of V: int8 tiles as loaded, fp16 tiles. (int8: few enough that the scales of SR key
    // tiles cover those on their way; at head dim 128 a second fp16 K tile is worth more than a second raw one.)
    static constexpr int RAWS = SRC != SRC_I8 ? 0 : D == 128 ? 1 : 2;
    static constexpr int FIT = (BUDGET - 2 * QTILE - 2 * RAWS * RAW) / ITEM;
    static constexpr int MOST = SRC == SRC_I8 ? 6 : CU_CLEAN;
    static constexpr int STAGES = FIT > MOST ? MOST : FIT;
    static constexpr int NK = STAGES / 2, NV = STAGES - NK;
    static constexpr int SOFT = 8, HELPER0 = 12, HELPERS = 4, THREADS = 512;
    // registers per thread after the split; the launch gives 65536 / THREADS, rounded down to 8
    static constexpr int REGS_LAUNCH = 65536 / THREADS / 8 * 8;
    static constexpr int REGS_REST = 64;
    static constexpr int REGS_SOFT = (THREADS * REGS_LAUNCH - (THREADS - 32 * SOFT) * REGS_REST) / (32 * SOFT) / 8 * 8;
    // Tensor-memory columns. fp16 probabilities have their own, so that a tile's next scores need not wait
    // for its value product; split ones lie over their scores. O of tile t is at O_COL + D t.
    static constexpr bool ALIAS = QF32;
    static constexpr int SBUFS = ALIAS || D == 64 ? 2 : 1;    // score buffers: the tiles', or one that they share
    static constexpr int O_COL = ALIAS ? 256 : 128 * SBUFS + 128;
    static_assert(O_COL + 2 * D <= 512, "tensor memory");
    // int8: key tiles whose scales are kept, enough that the ring holds no key tile up. (A query tile can fall
    // several key tiles behind the other one, over units that only that one has rows in, so a slot is
    // written when both are through with what it held.)
    static constexpr int SR = SRC != SRC_I8 ? 0 : QF32 && D == 128 ? 4 : 8;
    static_assert(SRC != SRC_I8 || RAWS + NK + 2 <= SR, "scale ring");
    static constexpr size_t Q_OFF = 0;
    static constexpr size_t KV_OFF = 2 * QTILE;
    static constexpr size_t RAW_OFF = KV_OFF + size_t(STAGES) * ITEM;  // (K's stages, then V's)
    static constexpr size_t BAR_OFF = RAW_OFF + size_t(2 * RAWS) * RAW;
    static constexpr int NBARS = 2 * STAGES + 4 * RAWS + 11 + CU_CLEAN + 2 * CU_RING + SR;
    static constexpr size_t UNIT_OFF = kvb_align_up(BAR_OFF + 8 * NBARS, 64);
    static constexpr size_t SCALE_OFF = UNIT_OFF + 64 * CU_RING;           // [SR tiles][K, V][16 pages]
    // [SR tiles][16 pages]: the largest biased exponent of a finite V scale up to each page
    static constexpr size_t VMAX_OFF = SCALE_OFF + (RAWS ? SR * 2 * 16 * 4 : 0);
    static constexpr size_t MISC_OFF = kvb_align_up(VMAX_OFF + (RAWS ? SR * 16 : 0), 16);
    static constexpr size_t SMEM = MISC_OFF + 16 + 4 * CU_CLEAN + 1024;
    static_assert(NK >= 1 && NV >= 1 && SMEM <= 227 * 1024, "shared memory budget");
    static_assert(KV_OFF % 1024 == 0 && RAW_OFF % 1024 == 0, "swizzled tiles need 1024-byte alignment");
};

// A unit as the roles share it.
struct RingUnit {
    ChunkUnit u;
    int t0;         // first key tile
    int nt[2];      // key tiles of the two query tiles
    int slot;       // where its partial result goes; -1: the unit is whole
    int odd;        // a seen value was not finite (set by the cleaning warps)
    int bad;        // first position whose block id was refused (the producers' minimum): the rows that see it are
                    // NaN. A query tile with fewer key tiles may read it while a later one's is set: no row of it
                    // sees that position
};
static_assert(sizeof(RingUnit) <= 64, "ring entry");

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Largest of three, NaN if one is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
__device__ __forceinline__ float fmaxf_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ float fminf_nan(float a, float b) {
    float y;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// Two fp32 operations per instruction.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t y;
    asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ void unpack2(uint64_t x, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t y;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(a), "l"(b), "l"(c));
    return y;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t y;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
    return y;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t y;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
    return y;
}

// 2^x of a pair on the FMA pipe: x = n + r with n the nearest integer and r in [-1/2, 1/2], 2^r by its
// minimax polynomial of degree 4 (fitted to the relative error, 2.6e-6, far below the fp16 rounding that
// follows), times 2^n. x + 1.5 * 2^23 + 127 holds n + 127, 2^n's exponent, in its low bits. x is taken into
// [-127, 127], where that is 0 (a factor of 0) to 254: with a reference that a key tile has left far behind x has
// no bound, and 2^127 makes the sum raise the reference as infinity would. NaN stays NaN.
__device__ __forceinline__ void exp2_poly2(uint64_t x, float& a, float& b) {
    unpack2(x, a, b);
    x = pack2(fminf_nan(fmaxf_nan(a, -127.f), 127.f), fminf_nan(fmaxf_nan(b, -127.f), 127.f));
    const uint64_t magic = pack2(12583039.f, 12583039.f), minus = pack2(-12583039.f, -12583039.f);
    const uint64_t n = add2(x, magic);
    const uint64_t r = fma2(add2(n, minus), pack2(-1.f, -1.f), x);
    uint64_t y = fma2(r, pack2(0.009570102207362652f, 0.009570102207362652f), pack2(0.05591785907745361f, 0.05591785907745361f));
    y = fma2(y, r, pack2(0.240247443318367f, 0.240247443318367f));
    y = fma2(y, r, pack2(0.6931217908859253f, 0.6931217908859253f));
    y = fma2(y, r, pack2(0.9999992847442627f, 0.9999992847442627f));
    float na, nb;
    unpack2(n, na, nb);
    y = mul2(y, pack2(__uint_as_float(__float_as_uint(na) << 23), __uint_as_float(__float_as_uint(nb) << 23)));
    unpack2(y, a, b);
}

// 32 bytes in one store: each thread writes a row of its own, and its rows lie lines apart, so the number of
// store instructions is what the outputs cost.
__device__ __forceinline__ void store32(void* dst, const uint32_t* r) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

// Pins the loaded values behind the wait that makes them valid.
template <int N>
__device__ __forceinline__ void pin(uint32_t* r) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}

__device__ __forceinline__ bool finite_half(__half h) { return (__half_as_ushort(h) & 0x7c00u) != 0x7c00u; }

template <int SRC, bool QF32, int D>
__global__ void __launch_bounds__((CCfg<SRC, QF32, D>::THREADS), 1)
    chunk_umma_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                      const __grid_constant__ CUtensorMap tmv, const __grid_constant__ ChunkParams p) {
    using C = CCfg<SRC, QF32, D>;
    using QT = typename std::conditional<QF32, float, __half>::type;
    constexpr int NSUB = C::NSUB, NK = C::NK, NV = C::NV, RAWS = C::RAWS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = smem_u32(smem);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
    uint64_t* k_full = bars;             // [NK] key tile ready for the products
    uint64_t* v_full = k_full + NK;      // [NV] value tile ready
    uint64_t* k_empty = v_full + NV;     // [NK] its products are done
    uint64_t* v_empty = k_empty + NK;
    uint64_t* rk_full = v_empty + NV;    // [RAWS] int8 key tile loaded
    uint64_t* rv_full = rk_full + RAWS;
    uint64_t* rk_empty = rv_full + RAWS;  // [RAWS] ... and converted
    uint64_t* rv_empty = rk_empty + RAWS;
    uint64_t* q_full = rv_empty + RAWS;  // [2] query tile in shared memory
    uint64_t* q_empty = q_full + 2;      // both query tiles' score products are done
    uint64_t* s_full = q_empty + 1;      // [2] scores of the tile ready
    uint64_t* s_free = s_full + 2;       // [SBUFS] scores read into registers (not with ALIAS)
    uint64_t* p_full = s_free + 2;       // [2] probabilities written, O scaled
    uint64_t* pv_done = p_full + 2;      // [2] a value product done
    uint64_t* dirty_full = pv_done + 2;   // [CU_CLEAN] a value tile loaded that passes the cleaning warps first
    uint64_t* r_full = dirty_full + CU_CLEAN;  // [CU_RING] unit published
    uint64_t* r_empty = r_full + CU_RING;
    uint64_t* sc_free = r_empty + CU_RING;  // [SR] int8: both softmax groups are through with the slot's scales
    auto ring = [&](int e) -> RingUnit& { return *reinterpret_cast<RingUnit*>(smem + C::UNIT_OFF + 64 * (e % CU_RING)); };
    float* s_scale = reinterpret_cast<float*>(smem + C::SCALE_OFF);
    uint8_t* s_vmax = smem + C::VMAX_OFF;
    volatile int* s_abort = reinterpret_cast<volatile int*>(smem + C::MISC_OFF);
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + C::MISC_OFF + 8);
    unsigned* s_clean = reinterpret_cast<unsigned*>(smem + C::MISC_OFF + 16);  // [CU_CLEAN] cleaning warps done
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (warp == 0) {
        for (int i = lane; i < C::NBARS; i += 32) {
            uint64_t* b = bars + i;
            uint32_t n = 1;
            if (b < k_empty) n = SRC == SRC_I8 ? C::HELPERS / 2 : 1;
            else if (b >= rk_empty && b < q_full) n = C::HELPERS / 2;
            else if (b >= q_full && b < q_empty) n = QF32 ? C::SOFT / 2 : 1;
            else if (b >= s_free && b < pv_done) n = C::SOFT / 2;
            else if (b >= sc_free) n = C::SOFT;
            else if (b >= r_empty) n = (C::ALIAS ? 2 : 3) + C::SOFT + C::HELPERS;  // V producer, issuers, the rest
            mbar_init(b, n);
        }
        if (lane == 0) {
            *s_abort = 0;
            for (int i = 0; i < CU_CLEAN; ++i) s_clean[i] = 0;
        }
        fence_mbarrier_init();
    }
    if (warp == 10) {
        tc_alloc(s_tmem, 512);
        tc_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    pdl_wait();
    pdl_trigger();

    // This CTA's part of the work: the whole line's length, and the sequence that the part begins in. Up to 32
    // sequences are added up by one warp, more by all threads. (In the stages' memory, which nothing loads
    // into yet.)
    long long* s_sum = reinterpret_cast<long long*>(smem + C::KV_OFF);
    volatile long long* s_begin = s_sum + C::THREADS;  // sequence, place in it, the line
    auto seq_cost = [&](int b) {
        const ChunkSeq s = chunk_seq(p, b);
        return p.Hkv * cost_upto(p, s, seq_units(p, s));
    };
    auto parts_of = [&](long long line) { return min((long long)p.ctas, max(1ll, line / CU_COST_LEAST)); };
    auto warp_sums = [&](long long x) {  // inclusive, over the lanes
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        return x;
    };
    if (p.B <= 32) {
        if (warp == 0) {
            const long long mine = lane < p.B ? seq_cost(lane) : 0, upto = warp_sums(mine);
            const long long total = __shfl_sync(0xffffffffu, upto, 31), n = parts_of(total);
            const long long at = (blockIdx.x >= n ? total : total * blockIdx.x / n) - (upto - mine);
            if (lane == 0) {
                s_begin[0] = p.B;
                s_begin[2] = total;
            }
            __syncwarp();
            if (at >= 0 && at < mine) {
                s_begin[0] = lane;
                s_begin[1] = at;
            }
        }
    } else {
        const int per = (p.B + C::THREADS - 1) / C::THREADS, used = (p.B + per - 1) / per;
        const int b0 = min(p.B, tid * per), b1 = min(p.B, b0 + per);
        long long mine = 0;
        for (int b = b0; b < b1; ++b) mine += seq_cost(b);
        s_sum[tid] = mine;
        if (tid == 0) s_begin[0] = p.B;
        __syncthreads();
        if (warp == 0) {  // exclusive sums, and the total behind them
            long long carry = 0;
            for (int i = lane; i < (used + 31) / 32 * 32; i += 32) {
                const long long v = s_sum[i], x = warp_sums(v);
                s_sum[i] = carry + x - v;
                carry += __shfl_sync(0xffffffffu, x, 31);
            }
            if (lane == 0) s_begin[2] = carry;
        }
        __syncthreads();
        const long long total = s_begin[2], n = parts_of(total);
        long long at = (blockIdx.x >= n ? total : total * blockIdx.x / n) - s_sum[tid];
        if (at >= 0 && at < mine) {
            int b = b0;
            for (; b < b1; ++b) {
                const long long w = seq_cost(b);
                if (at < w) break;
                at -= w;
            }
            s_begin[0] = b;
            s_begin[1] = at;
        }
    }
    __syncthreads();
    const long long line = s_begin[2], parts = parts_of(line);
    auto part_begin = [&](long long c) { return c >= parts ? line : line * c / parts; };
    const long long my_begin = part_begin(blockIdx.x), my_end = part_begin(blockIdx.x + 1ll);
    const int first_seq = int(s_begin[0]);
    const long long first_at = s_begin[1];
    fence_proxy_async_smem();
    __syncthreads();  // read before the stages are loaded

    // False once a wait has given up (here, or elsewhere in the CTA where this one would block).
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (mbar_try_wait(bar, parity & 1)) return true;
        if (!*s_abort && mbar_wait_bounded(bar, parity & 1, s_abort)) return true;
        *s_abort = 1;
        return false;
    };
    auto stop = [&]() { return __any_sync(0xffffffffu, *s_abort) != 0; };  // the same answer in a whole warp

    if (warp < C::SOFT) {
        // ---------------------------------------------------------------- softmax, one thread per query row
        reg_alloc<C::REGS_SOFT>();
        const int t = warp >> 2;
        const int r = tid & 127;  // row of the tile
        const uint32_t lanes = uint32_t(warp & 3) << 21;  // this warp's quarter of the tensor-memory lanes
        const uint32_t ts = tmem + lanes + 128 * (t % C::SBUFS), to = tmem + lanes + C::O_COL + D * t;
        const uint32_t tp = C::ALIAS ? ts : tmem + lanes + 128 * C::SBUFS + 64 * t;
        const int tok = r / p.G, head = r % p.G;
        const int lp = SRC == SRC_I8 ? __ffs(p.page) - 1 : 0;
        uint32_t ns = 0, np = 0;  // scores taken, probabilities handed over
        uint32_t tiles = 0;       // key tiles of the CTA so far (int8 scale ring)
        constexpr int FOLD = QF32 ? CU_FOLD_F32 : CU_FOLD_F16;
        float4* fold = reinterpret_cast<float4*>(p.fold) + (size_t)(2 * blockIdx.x + t) * (D / 4) * 128 + r;
        for (int e = 0;; ++e) {
            wait(&r_full[e % CU_RING], e / CU_RING);
            if (stop()) break;
            const RingUnit& R = ring(e);
            const ChunkUnit u = R.u;
            const int nt = R.nt[t], nall = max(R.nt[0], R.nt[1]), kt0 = R.t0, slot = R.slot;
            if (u.state < 0) break;
            auto leave = [&]() {
                __syncwarp();
                if (lane == 0) mbar_arrive(&r_empty[e % CU_RING]);
            };
            // The unit's key tiles from j on, which only the other query tile has. (One turn of the ring at a
            // time: an arrival counts for the phase that is open.)
            auto pass = [&](int j) {
                if constexpr (SRC == SRC_I8) {
                    for (; j < nall && !stop(); ++j) {
                        const uint32_t i = tiles + j;
                        if (i >= C::SR) wait(&sc_free[i % C::SR], i / C::SR - 1);
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sc_free[i % C::SR]);
                    }
                }
                tiles += nall;
            };
            if (u.state == 2) {
                if (warp < 4) chunk_refuse<QT, D>(p, u, r, 128);
                leave();
                continue;
            }
            const int tt = t * p.tile_tokens;              // first token of the tile in the unit
            const int cnt = min(u.n - tt, p.tile_tokens);  // its tokens
            if (cnt <= 0) {
                pass(0);
                leave();
                continue;
            }
            const bool live = tok < cnt;
            const int my = min(tok, cnt - 1);
            const int limit = u.pos0 + tt + my + 1;        // keys that this row sees
            const int all_see = u.pos0 + tt + 1;           // keys that every row of the tile sees
            const long long qrow = u.row0 + tt + my;
            const int h = u.kvh * p.G + head;
            float f = p.q_scale;
            if constexpr (QF32) {
                if (nt > 0) {
                    // this row's query, split; the tile's previous scores are done (these warps waited for them)
                    const float4* q4 = reinterpret_cast<const float4*>(
                        static_cast<const float*>(p.q) + qrow * p.q_stride + (long long)h * D);
                    float amax = 0.f;
#pragma unroll 8
                    for (int i = 0; i < D / 4; ++i) {
                        const float4 a = q4[i];
                        amax = fmaxf(amax, max4(make_float4(fabsf(a.x), fabsf(a.y), fabsf(a.z), fabsf(a.w))));
                    }
                    // 2^-x amax in [1, 2) for a normal amax: exact, and the halves keep their 22 bits
                    int x = int(__float_as_uint(amax) >> 23) - 127;
                    x = amax > 0.f && x < 128 ? min(max(x, -100), 126) : 0;
                    const float down = __uint_as_float(uint32_t(127 - x) << 23);
                    f *= __uint_as_float(uint32_t(127 + x) << 23);
                    uint8_t* qs = smem + C::Q_OFF + t * C::QTILE;
#pragma unroll 4
                    for (int i = 0; i < D / 8; ++i) {
                        const float4 a = q4[2 * i], b = q4[2 * i + 1];
                        uint4 hi, lo;
                        split_hi_lo(a.x * down, a.y * down, hi.x, lo.x);
                        split_hi_lo(a.z * down, a.w * down, hi.y, lo.y);
                        split_hi_lo(b.x * down, b.y * down, hi.z, lo.z);
                        split_hi_lo(b.z * down, b.w * down, hi.w, lo.w);
                        const uint32_t off = (i / 8) * CU_SUB + swz_off(r, (i % 8) * 16);
                        *reinterpret_cast<uint4*>(qs + off) = hi;
                        *reinterpret_cast<uint4*>(qs + NSUB * CU_SUB + off) = lo;
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&q_full[t]);
                }
            }
            float ref = -INFINITY;  // probabilities are 2^(f s - ref)
            const float most = live ? CU_MOST : INFINITY;  // rows of no token hold anything: they move no reference
            // Until a row has a reference (every score so far was -inf) the first finite score has to move it: with
            // the largest number in its place such a score's probability is inf, and that of -inf 0.
            auto minus_ref = [&]() { return ref == -INFINITY ? 3.402823466e38f : -ref; };
            float l = 0.f;
            float vexp = 0.f;       // int8: 2^-e, probabilities times the value scales times this; 0: not set yet
            float older = 1.f;      // what the folded sum has to be scaled by
            int folds = 0;
            // every value product of this tile so far is done
            auto settled = [&]() {
                if (np > 0) wait(&pv_done[t], np - 1);
                tc_fence_after();
            };
            // O (complete up to here) and the folded sum times `scale`
            auto rescale = [&](float scale) {
                older *= scale;
                settled();
#pragma unroll 1
                for (int c = 0; c < D; c += 16) {
                    uint32_t o[16];
                    tc_ld16(to + c, o);
                    tc_wait_ld();
                    pin<16>(o);
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * scale);
                    tc_st16(to + c, o);
                }
                tc_wait_st();  // a second call for the same key tile loads what this one stored
            };
            // fp32 queries on fp16 pages: the scores that are NaN among 32 of a key tile once more, in fp32 (on keys
            // with an infinite component, so that their scale does not matter: -inf, +inf or NaN).
            auto rescore = [&](int k0, int c0) {
                const float* qr = static_cast<const float*>(p.q) + qrow * p.q_stride + (long long)h * D;
#pragma unroll 1
                for (int c = c0; c < c0 + 32; ++c) {
                    uint32_t x = tc_ld1(ts + c);
                    tc_wait_ld();
                    pin<1>(&x);
                    const bool odd = __uint_as_float(x) != __uint_as_float(x) && k0 + c < limit;
                    const __half* kr = odd ? chunk_row<__half>(p, u, p.k, p.k_stride, k0 + c, D) : nullptr;
                    if (kr) {
                        float y = 0.f;
#pragma unroll 1
                        for (int i = 0; i < D; ++i) y = fmaf(qr[i], __half2float(kr[i]), y);
                        x = __float_as_uint(y);
                    }
                    __syncwarp();
                    tc_st1(ts + c, x);
                }
                tc_wait_st();
            };
            bool lost = false;
            for (int j = 0; j < nt; ++j) {
                const int k0 = (kt0 + j) * CU_ROWS;  // first key
                const bool masked = k0 + CU_ROWS > all_see;
                const float* scales = s_scale + (tiles + j) % std::max(C::SR, 1) * 32;
                lost = __any_sync(0xffffffffu, !wait(&s_full[t], ns++)) != 0;
                if (lost) break;
                tc_fence_after();
                // What O needs before the reference: waits for the value product before. The issuer reaches that
                // one only after other scores, so with a shared score buffer this comes after s_free.
                auto settle_outputs = [&]() {
                    if (j > 0 && j % FOLD == 0) {
                        // the next product starts O anew
                        settled();
                        constexpr int FW = C::ALIAS ? 32 : 16;  // columns at a time (16 beside a tile's scores)
                        const bool plain = __all_sync(0xffffffffu, older == 1.f);
#pragma unroll 1
                        for (int c = 0; c < D; c += FW) {
                            uint32_t o[FW];
                            if constexpr (FW == 32) tc_ld32(to + c, o);
                            else tc_ld16(to + c, o);
                            tc_wait_ld();
                            pin<FW>(o);
                            float4* at = fold + (c / 4) * 128;
#pragma unroll
                            for (int i = 0; i < FW / 4; ++i, at += 128) {
                                float4 x = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                                                       __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
                                if (folds == 0) {
                                    __stcg(at, x);
                                } else if (plain) {
                                    asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(at), "f"(x.x), "f"(x.y),
                                                 "f"(x.z), "f"(x.w)
                                                 : "memory");
                                } else {
                                    const float4 y = __ldcg(at);
                                    x.x = fmaf(y.x, older, x.x), x.y = fmaf(y.y, older, x.y);
                                    x.z = fmaf(y.z, older, x.z), x.w = fmaf(y.w, older, x.w);
                                    __stcg(at, x);
                                }
                            }
                        }
                        ++folds;
                        older = 1.f;
                    }
                    if constexpr (SRC == SRC_I8) {
                        // the largest value scale among the pages that this row sees (a larger one behind them would
                        // push the row's probabilities out of fp16's range), down to a power of two
                        const int last = masked ? (min(limit - k0, CU_ROWS) - 1) >> lp : 15;
                        const int vm = last >= 0 ? s_vmax[(tiles + j) % C::SR * 16 + last] : 0;
                        const bool move = vexp == 0.f || __uint_as_float(uint32_t(vm) << 23) * vexp > 1.f;
                        // (the rows differ in masked tiles only, which are a unit's last)
                        if (masked ? __any_sync(0xffffffffu, move) != 0 : move) {
                            // times the scale in [0.5, 1)
                            const float ve = __uint_as_float(uint32_t(253 - min(max(vm, 27), 252)) << 23);
                            if (j > 0) rescale(move ? ve / vexp : 1.f);
                            if (move) vexp = ve;
                        }
                    }
                };
                float sum = 0.f;
                if constexpr (C::ALIAS) {
                    // 32 keys at a time: hi, then lo halves, 16 columns each, over the scores they came from. The
                    // reference is a whole number here, so that probabilities already written can follow it
                    // exactly.
                    settle_outputs();
                    settled();
#pragma unroll 1
                    for (int c0 = 0; c0 < CU_ROWS; c0 += 32) {
                        uint32_t s[32], pr[32];
                        float part, top;
#pragma unroll 1
                        for (bool again = false;; again = true) {
                            tc_ld32(ts + c0, s);
                            tc_wait_ld();
                            pin<32>(s);
                            if constexpr (SRC == SRC_I8) {
#pragma unroll
                                for (int c = 0; c < 32; c += 8) {
                                    const float ks = scales[(c0 + c) >> lp];
#pragma unroll
                                    for (int i = 0; i < 8; ++i) s[c + i] = __float_as_uint(__uint_as_float(s[c + i]) * ks);
                                }
                            }
                            const int lim = limit - k0 - c0;
                            if (masked) {
                                const uint32_t sees = lim >= 32 ? ~0u : lim <= 0 ? 0u : (1u << lim) - 1u;
#pragma unroll
                                for (int c = 0; c < 32; ++c)
                                    if (!(sees >> c & 1u)) s[c] = 0xff800000u;  // -inf
                            }
                            part = top = 0.f;
                            bool raise = j == 0 && c0 == 0;
                            for (;;) {
                                if (raise) {
                                    tc_wait_st();  // the tile's probabilities so far are loaded again below
                                    float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
                                    for (int i = 0; i < 32; i += 4) {
                                        m0 = max3_nan(m0, __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
                                        m1 = max3_nan(m1, __uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
                                    }
                                    top = fmaxf_nan(m0, m1) * f;
                                    const float up = ceilf(top) - CU_SHIFT;
                                    float scale = 1.f;
                                    if (up > ref) {
                                        scale = ref == -INFINITY ? 0.f : ex2(ref - up);
                                        ref = up;
                                            l *= scale;
                                        sum *= scale;
                                    }
                                    if (j > 0) rescale(scale);
                                    const __half2 by = __float2half2_rn(scale);  // a power of two, or 0 when none is left
#pragma unroll 1
                                    for (int c = 0; c < c0; c += 16) {
                                        uint32_t w[16];
                                        tc_ld16(tp + c, w);
                                        tc_wait_ld();
                                        pin<16>(w);
#pragma unroll
                                        for (int i = 0; i < 16; ++i) w[i] = h2_as_u32(__hmul2(u32_as_h2(w[i]), by));
                                        tc_st16(tp + c, w);
                                    }
                                }
                                const float base = minus_ref();
                                const uint64_t f2 = pack2(f, f), b2 = pack2(base, base);
                                uint64_t l0 = 0, l1 = 0;
                                float vs = 0.f;
#pragma unroll
                                for (int i = 0; i < 32; i += 2) {
                                    float a, b;
                                    unpack2(fma2(pack2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), f2, b2), a, b);
                                    a = ex2(a);
                                    b = ex2(b);
                                    if (i & 2) l1 = add2(l1, pack2(a, b));
                                    else l0 = add2(l0, pack2(a, b));
                                    if constexpr (SRC == SRC_I8) {
                                        if (i % 8 == 0) vs = scales[16 + ((c0 + i) >> lp)] * vexp;  // pages of 8 tokens at least
                                        a *= vs;
                                        b *= vs;
                                        if (masked) {  // the scale of a page that this row does not see may be anything
                                            if (i >= lim) a = 0.f;
                                            if (i + 1 >= lim) b = 0.f;
                                        }
                                    }
                                    split_hi_lo(a, b, pr[i / 2], pr[16 + i / 2]);
                                }
                                float a, b;
                                unpack2(add2(l0, l1), a, b);
                                part = a + b;
                                if (raise || !__any_sync(0xffffffffu, part > most)) break;
                                raise = true;
                            }
                            // A NaN that is the row's first may come from an infinite key and the two parts of a
                            // query, of which one may be 0 or of the other sign.
                            if (SRC != SRC_F16 || again ||
                                !__any_sync(0xffffffffu, part != part && sum == sum && l == l))
                                break;
                            rescore(k0, c0);
                        }
                        tc_st32(tp + c0, pr);
                        sum += top < INFINITY ? part : __int_as_float(0x7fc00000);
                    }
                } else {
                    // the scores move to registers at once, and their buffer is free for the next ones
                    uint32_t s[CU_ROWS];
#pragma unroll
                    for (int c0 = 0; c0 < CU_ROWS; c0 += 32) tc_ld32(ts + c0, s + c0);
                    tc_wait_ld();
                    pin<CU_ROWS>(s);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s_free[t % C::SBUFS]);
                    settle_outputs();
                    // int8: the scale of a key's page is in the factor of its score, but for a masked tile's, whose
                    // scores have it before -inf takes their places.
                    auto factor = [&](int c) { return SRC == SRC_I8 && !masked ? f * scales[c >> lp] : f; };
                    if (masked) {
                        if constexpr (SRC == SRC_I8) {
#pragma unroll
                            for (int c = 0; c < CU_ROWS; c += 8) {
                                const float ks = scales[c >> lp];  // (pages of 128 tokens or more: one)
#pragma unroll
                                for (int i = 0; i < 8; ++i) s[c + i] = __float_as_uint(__uint_as_float(s[c + i]) * ks);
                            }
                        }
                        const int lim = limit - k0;
#pragma unroll
                        for (int c0 = 0; c0 < CU_ROWS; c0 += 32) {
                            // one bit a key, so that a few instructions make the predicates
                            const uint32_t sees = lim - c0 >= 32 ? ~0u : lim - c0 <= 0 ? 0u : (1u << (lim - c0)) - 1u;
#pragma unroll
                            for (int c = 0; c < 32; ++c)
                                if (!(sees >> c & 1u)) s[c0 + c] = 0xff800000u;  // -inf
                        }
                    }
                    settled();  // the product that reads the probabilities before these
                    // The probabilities to tensor memory; their sum.
                    auto probabilities = [&]() {
                        const float base = minus_ref();
                        const uint64_t b2 = pack2(base, base);
                        uint64_t f2 = pack2(f, f), v2 = 0;
                        uint64_t l0 = 0, l1 = 0;
#pragma unroll
                        for (int c0 = 0; c0 < CU_ROWS; c0 += 32) {
                            uint32_t pr[16];
#pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                if (SRC == SRC_I8 && i % 8 == 0) {  // pages of 8 tokens at least
                                    const float fk = factor(c0 + i), vs = scales[16 + ((c0 + i) >> lp)] * vexp;
                                    f2 = pack2(fk, fk);
                                    v2 = pack2(vs, vs);
                                }
                                const uint64_t x =
                                    fma2(pack2(__uint_as_float(s[c0 + i]), __uint_as_float(s[c0 + i + 1])), f2, b2);
                                float a, b;
                                if (CU_POLY_OF<D> > 0 && i / 2 % std::max(CU_POLY_OF<D>, 1) == 0) {
                                    exp2_poly2(x, a, b);
                                } else {
                                    unpack2(x, a, b);
                                    a = ex2(a);
                                    b = ex2(b);
                                }
                                if (i & 2) l1 = add2(l1, pack2(a, b));
                                else l0 = add2(l0, pack2(a, b));
                                if constexpr (SRC == SRC_I8) unpack2(mul2(pack2(a, b), v2), a, b);
                                pr[i / 2] = h2_as_u32(__floats2half2_rn(a, b));
                            }
                            if (SRC == SRC_I8 && masked) {  // the scale of a page that this row does not see may be anything
                                const int n = limit - k0 - c0;
                                const uint32_t sees = n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u;
#pragma unroll
                                for (int i = 0; i < 16; ++i)
                                    pr[i] &= (sees >> 2 * i & 1u ? 0xffffu : 0u) | (sees >> (2 * i + 1) & 1u ? 0xffff0000u : 0u);
                            }
                            tc_st16(tp + c0 / 2, pr);
                        }
                        float a, b;
                        unpack2(add2(l0, l1), a, b);
                        return a + b;
                    };
                    // With the reference so far first. No probability is above their sum, so a sum in bounds needs
                    // no maximum (a NaN makes the row NaN as it is). Otherwise, and until there is a reference, it
                    // rises to the highest score, O and l follow, and the probabilities are computed with that. (One copy of their code: the instruction cache holds little more than the loop.)
                    float top = 0.f;
                    bool raise = j == 0;
                    for (;;) {
                        if (raise) {
                            tc_wait_st();  // the probabilities stored so far are stored again
                            float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
                            for (int i = 0; i < CU_ROWS; i += 4) {
                                const float fk = SRC == SRC_I8 ? factor(i) : 1.f;
                                m0 = max3_nan(m0, __uint_as_float(s[i]) * fk, __uint_as_float(s[i + 1]) * fk);
                                m1 = max3_nan(m1, __uint_as_float(s[i + 2]) * fk, __uint_as_float(s[i + 3]) * fk);
                            }
                            top = fmaxf_nan(m0, m1) * (SRC == SRC_I8 ? 1.f : f) - CU_SHIFT;
                            float scale = 1.f;
                            if (top > ref) {
                                scale = ref == -INFINITY ? 0.f : ex2(ref - top);
                                ref = top;
                                l *= scale;
                            }
                            if (j > 0) rescale(scale);
                        }
                        sum = probabilities();
                        if (raise || !__any_sync(0xffffffffu, sum > most)) break;
                        raise = true;
                    }
                    if (!(top < INFINITY)) sum = __int_as_float(0x7fc00000);  // a NaN or +inf score: the row is NaN
                }
                l += sum;
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&p_full[t]);
                    if constexpr (SRC == SRC_I8) mbar_arrive(&sc_free[(tiles + j) % C::SR]);
                }
                ++np;
            }
            if (lost) break;
            pass(nt);
            settled();
            const volatile RingUnit& V = R;
            const bool bad = V.bad < limit, odd = V.odd != 0;
            if (__any_sync(0xffffffffu, bad) && lane == 0) raise_error(p.error_flag, KVB_DEVERR_BLOCK);
            float inv = bad ? __int_as_float(0x7fc00000) : slot >= 0 && l == 0.f ? 0.f : 1.f / l;
            const size_t row = (size_t)qrow * p.H + h;
            const size_t at = ((size_t)slot * 2 + t) * CU_ROWS + r;
            if (slot >= 0 && live) p.part_ml[at] = make_float2(ref, bad ? inv : l);
            if constexpr (SRC == SRC_I8) inv = vexp != 0.f ? inv / vexp : inv;
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                __syncwarp();
                if (nt > 0) {
                    tc_ld32(to + c, o);
                    tc_wait_ld();
                    pin<32>(o);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0;
                }
                if (folds > 0) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float4 x = __ldcg(fold + (c / 4 + i) * 128);
                        o[4 * i] = __float_as_uint(fmaf(x.x, older, __uint_as_float(o[4 * i])));
                        o[4 * i + 1] = __float_as_uint(fmaf(x.y, older, __uint_as_float(o[4 * i + 1])));
                        o[4 * i + 2] = __float_as_uint(fmaf(x.z, older, __uint_as_float(o[4 * i + 2])));
                        o[4 * i + 3] = __float_as_uint(fmaf(x.w, older, __uint_as_float(o[4 * i + 3])));
                    }
                }
                if (SRC != SRC_I8 && odd && !bad && live) {
                    // (the tiles are cleaned from the first one that some row of the unit, not of this query
                    // tile, does not see in full)
                    const int first = max(kt0, (u.pos0 + 1) / CU_ROWS) * CU_ROWS;
                    for (int k = first; k < min(limit, (kt0 + nt) * CU_ROWS); ++k) {
                        const __half* v = chunk_row<__half>(p, u, p.v, p.v_stride, k, D) + c;
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (!finite_half(v[i])) o[i] = __float_as_uint(__uint_as_float(o[i]) + __half2float(v[i]));
                    }
                }
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * inv);
                if (!live) {
                    // a row of no token: nothing to store
                } else if (QF32 || slot >= 0) {
                    uint4* out = reinterpret_cast<uint4*>(slot >= 0 ? p.part_o + at * D + c
                                                                       : static_cast<float*>(p.out) + row * D + c);
#pragma unroll
                    for (int i = 0; i < 4; ++i) store32(out + 2 * i, o + 8 * i);
                } else {
                    uint4* out = reinterpret_cast<uint4*>(static_cast<__half*>(p.out) + row * D + c);
                    uint32_t h[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        h[i] = h2_as_u32(__floats2half2_rn(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1])));
                    store32(out, h);
                    store32(out + 2, h + 8);
                }
            }
            tc_fence_before();
            leave();
        }
    } else {
        reg_dealloc<C::REGS_REST>();
        // One K or V tile (key tile `tile` of unit u) into stage `st` of its kind, by a whole warp: this lane's
        // box is page (or 128 tokens of a larger page) `id`.
        const int bt = SRC == SRC_PACKED ? CU_ROWS : min(p.page, CU_ROWS);  // keys of a box
        auto box_id = [&](const ChunkUnit& u, int tile, int end) {
            const int k = tile * CU_ROWS + lane * bt;
            if (SRC == SRC_PACKED || tile >= end || lane * bt >= CU_ROWS || k >= u.keys) return -1;
            return __ldg(p.block_table + (size_t)u.b * p.max_blocks + k / p.page);
        };
        auto load_tile = [&](const ChunkUnit& u, int tile, int id, bool is_v, uint32_t st, uint64_t* done, RingUnit& R) {
            const int k = tile * CU_ROWS + lane * bt;
            const bool wanted = SRC != SRC_PACKED && lane * bt < CU_ROWS && k < u.keys;
            const bool ok = wanted && id >= 0 && id < p.num_blocks;
            if (wanted && !ok) atomicMin(&R.bad, k);
            // A refused page of fp16 rows is a box before the pool's first row, which loads as zeros (int8: its scales
            // are 0). What shared memory held before could move the reference of rows beside those that see it.
            const bool loads = SRC == SRC_I8 ? ok : wanted;
            const uint32_t boxes = SRC == SRC_PACKED ? 1 : __popc(__ballot_sync(0xffffffffu, loads));
            const uint32_t bytes = SRC == SRC_I8 ? uint32_t(bt) * D : uint32_t(bt) * 128 * NSUB;  // of a box
            const bool off = *s_abort != 0;
            if (lane == 0) {
                if (boxes && !off) mbar_arrive_expect_tx(done, boxes * bytes);
                else mbar_arrive(done);
            }
            if (__any_sync(0xffffffffu, off)) return;  // (lane 0 may have expected bytes: the waits give up too)
            if constexpr (SRC == SRC_I8) {
                if (ok)
                    bulk_load(smem + C::RAW_OFF + ((is_v ? RAWS : 0) + st) * C::RAW + lane * bytes,
                              static_cast<const int8_t*>(is_v ? p.v : p.k) +
                                  (((long long)id * p.Hkv + u.kvh) * p.page + k % p.page) * D,
                              bytes, done);
            } else {
                uint8_t* dst = smem + C::KV_OFF + ((is_v ? NK : 0) + st) * C::ITEM;
                const CUtensorMap* map = is_v ? &tmv : &tmk;
                if constexpr (SRC == SRC_PACKED) {
                    if (lane == 0)
#pragma unroll
                        for (int s = 0; s < NSUB; ++s)
                            tma_load_3d(dst + s * CU_SUB, map, done, 64 * s, u.kvh, u.kv0 + tile * CU_ROWS);
                } else if (loads) {
                    const int y = ok ? (id * p.Hkv + u.kvh) * p.page + k % p.page : -bt;
#pragma unroll
                    for (int s = 0; s < NSUB; ++s)
                        tma_load_2d(dst + s * CU_SUB + lane * bt * 128, map, done, 64 * s, y);
                }
            }
            __syncwarp();
        };
        if (warp == 8) {
            // ------------------------------------------------------------ scheduler, keys and queries
            uint32_t item = 0, published = 0;  // key tiles, units
            uint32_t qn = 0;                   // units whose queries were loaded
            auto publish = [&](const ChunkUnit& u, int2 range, int nt0, int nt1, int slot) {
                if (published >= CU_RING) wait(&r_empty[published % CU_RING], published / CU_RING - 1);
                __syncwarp();
                if (lane == 0) {
                    RingUnit& R = ring(published);
                    R.u = u;
                    R.t0 = range.x;
                    R.nt[0] = nt0;
                    R.nt[1] = nt1;
                    R.slot = slot;
                    R.odd = 0;
                    R.bad = 0x7fffffff;
                    mbar_arrive(&r_full[published % CU_RING]);
                }
                ++published;
            };
            ChunkPiece piece{0, 0, 0, -1, 0};
            long long place = my_begin, at = first_at;  // on the line; in the sequence
            ChunkSeq s{};
            int units = 0;
            long long w = 0;  // cost of one KV head of sequence b
            for (int b = first_seq, known = -1; b < p.B && place < my_end && !stop();) {
                if (b != known) {
                    known = b;
                    s = chunk_seq(p, b);
                    units = seq_units(p, s);
                    w = cost_upto(p, s, units);
                }
                if (at >= w * p.Hkv) {
                    at = 0;
                    ++b;
                    continue;
                }
                ChunkUnit u;
                u.b = b;
                u.kvh = int(at / w);
                const long long x = at - u.kvh * w;
                int k = 0, hi = units - 1;  // the unit: the last one that begins at or before x
                while (k < hi) {
                    const int mid = k + (hi - k + 1) / 2;
                    if (cost_upto(p, s, mid) <= x) k = mid;
                    else hi = mid - 1;
                }
                const long long u0 = cost_upto(p, s, k), uw = cost_upto(p, s, k + 1) - u0;
                const long long xa = x - u0, xb = min(uw, xa + (my_end - place));  // this CTA's part of the unit
                const long long unit_end = place + (uw - xa);
                place += xb - xa;
                at += xb - xa;
                u.split = 0;
                u.kv0 = s.c0;
                if (s.bad) {
                    u.state = 2;
                    u.row0 = s.c0;
                    u.n = s.n;
                    u.pos0 = u.keys = 0;
                    if (xa == 0) publish(u, make_int2(0, 0), 0, 0, -1);
                    continue;
                }
                u.state = 0;
                u.row0 = s.c0 + k * p.unit_tokens;
                u.n = min(p.unit_tokens, s.n - k * p.unit_tokens);
                u.pos0 = s.ctx + k * p.unit_tokens;
                u.keys = u.pos0 + u.n;
                const int nt_all = (u.keys + CU_ROWS - 1) / CU_ROWS;
                const int2 range = make_int2(cut_tile(xa, uw, nt_all), cut_tile(xb, uw, nt_all));
                if (range.x == range.y) continue;
                int slot = -1;
                if (range.x > 0) {
                    slot = 2 * blockIdx.x;
                    piece.head = 1;
                } else if (range.y < nt_all) {
                    slot = 2 * blockIdx.x + 1;
                    piece.kvh = u.kvh;
                    piece.row0 = u.row0;
                    piece.n = u.n;
                    long long c = blockIdx.x + 1;  // the last part that begins before the unit's end
                    while (c + 1 < parts && part_begin(c + 1) < unit_end) ++c;
                    piece.last = int(c);
                }
                const int n1 = u.n - p.tile_tokens;  // tokens of tile 1
                const int keys0 = u.pos0 + min(u.n, p.tile_tokens);
                const int nt0 = max(0, min(range.y, (keys0 + CU_ROWS - 1) / CU_ROWS) - range.x);
                const int nt1 = n1 > 0 ? range.y - range.x : 0;
                const int e = published;
                publish(u, range, nt0, nt1, slot);
                const int nj = max(nt0, nt1);
                if (nj == 0) continue;
                const int end_tile = range.x + nj;
                int id = box_id(u, range.x, end_tile);  // read a tile ahead
                for (int tile = range.x; tile < end_tile && !stop(); ++tile, ++item) {
                    const int next = box_id(u, tile + 1, end_tile);
                    if constexpr (SRC == SRC_I8) {
                        const uint32_t st = item % RAWS;
                        const bool ok = id >= 0 && id < p.num_blocks;
                        const float ks = ok ? __ldg(p.k_scale + (long long)id * p.Hkv + u.kvh) : 0.f;
                        const float vs = ok ? __ldg(p.v_scale + (long long)id * p.Hkv + u.kvh) : 0.f;
                        if (item >= RAWS) wait(&rk_empty[st], item / RAWS - 1);
                        if (item >= C::SR) wait(&sc_free[item % C::SR], item / C::SR - 1);
                        int vm = __float_as_uint(vs) >> 23 & 255;  // its exponent, of finite ones
                        vm = vm < 255 ? vm : 0;
#pragma unroll
                        for (int o = 1; o < 16; o <<= 1) {
                            const int x = __shfl_up_sync(0xffffffffu, vm, o);
                            if (lane >= o) vm = max(vm, x);
                        }
                        if (lane < 16) {
                            s_scale[item % C::SR * 32 + lane] = ks;
                            s_scale[item % C::SR * 32 + 16 + lane] = vs;
                            s_vmax[item % C::SR * 16 + lane] = uint8_t(vm);
                        }
                        __syncwarp();
                        load_tile(u, tile, id, false, st, &rk_full[st], ring(e));
                    } else {
                        const uint32_t st = item % NK;
                        if (item >= NK) wait(&k_empty[st], item / NK - 1);
                        __syncwarp();
                        load_tile(u, tile, id, false, st, &k_full[st], ring(e));
                    }
                    id = next;
                    if (!QF32 && tile == range.x) {
                        // the queries, once the unit before has used its own
                        if (qn > 0) wait(q_empty, qn - 1);
                        ++qn;
                        if (lane == 0 && !*s_abort) {
                            const uint32_t bytes = uint32_t(p.tile_tokens * p.G) * 128 * NSUB;
#pragma unroll
                            for (int t = 0; t < 2; ++t) {
                                if ((t ? nt1 : nt0) == 0) continue;
                                mbar_arrive_expect_tx(&q_full[t], bytes);
#pragma unroll
                                for (int s = 0; s < NSUB; ++s)
                                    tma_load_3d(smem + C::Q_OFF + t * C::QTILE + s * CU_SUB, &tmq, &q_full[t], 64 * s,
                                                u.kvh * p.G, u.row0 + t * p.tile_tokens);
                            }
                        }
                        __syncwarp();
                    }
                }
            }
            ChunkUnit end{};
            end.state = -1;
            publish(end, make_int2(0, 0), 0, 0, -1);
            if (lane == 0) p.pieces[blockIdx.x] = piece;
        } else if (warp == 9) {
            // ------------------------------------------------------------ values
            uint32_t item = 0, dirty_n = 0;  // value tiles, those that went to the cleaning warps
            for (int e = 0; !stop(); ++e) {
                wait(&r_full[e % CU_RING], e / CU_RING);
                RingUnit& R = ring(e);
                const ChunkUnit u = R.u;
                if (u.state < 0) break;
                const int end_tile = R.t0 + max(R.nt[0], R.nt[1]);
                const int dirty = (u.pos0 + 1) / CU_ROWS;  // values from this tile on pass the cleaning warps
                int tile = R.t0, id = box_id(u, tile, end_tile);
                for (; tile < end_tile && !stop(); ++tile, ++item) {
                    const int next = box_id(u, tile + 1, end_tile);
                    if constexpr (SRC == SRC_I8) {
                        const uint32_t st = item % RAWS;
                        if (item >= RAWS) wait(&rv_empty[st], item / RAWS - 1);
                        __syncwarp();
                        load_tile(u, tile, id, true, st, &rv_full[st], R);
                    } else {
                        const uint32_t st = item % NV;
                        if (item >= NV) wait(&v_empty[st], item / NV - 1);
                        __syncwarp();
                        load_tile(u, tile, id, true, st, tile >= dirty ? &dirty_full[dirty_n++ % CU_CLEAN] : &v_full[st], R);
                    }
                    id = next;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&r_empty[e % CU_RING]);
            }
        } else if (warp == 10 || (warp == 11 && !C::ALIAS)) {
            // ------------------------------------------------------------ products
            if (tc_elect()) {
                constexpr uint32_t id_s = instr_desc(1, 0, 0, 0, 0, 128, 128);
                constexpr uint32_t id_o = instr_desc(1, 0, 0, 0, 1, D, 128);
                constexpr int FOLD = QF32 ? CU_FOLD_F32 : CU_FOLD_F16;
                // descriptors of the first stage; a byte offset of o adds o / 16
                const uint64_t kd = smem_desc(sbase + uint32_t(C::KV_OFF), 16, 1024);
                const uint64_t vd = smem_desc(sbase + uint32_t(C::KV_OFF + NK * C::ITEM), CU_SUB, 1024);
                const uint64_t qd = smem_desc(sbase + uint32_t(C::Q_OFF), 16, 1024);
                uint32_t item = 0;                // key tiles before the unit (and value tiles)
                uint32_t nq0 = 0, nq1 = 0, np0 = 0, np1 = 0, nb0 = 0, nb1 = 0;  // uses of each barrier
                auto scores = [&](int t, uint32_t it) {
                    if constexpr (!C::ALIAS) {  // the buffer's scores before these were read
                        uint32_t& nb = t % C::SBUFS ? nb1 : nb0;
                        if (nb > 0) wait(&s_free[t % C::SBUFS], nb - 1);
                        ++nb;
                    }
                    tc_fence_after();
                    const uint64_t k = kd + (it % NK) * (C::ITEM / 16), q = qd + t * (C::QTILE / 16);
                    // (rolled where the descriptors of both halves would spill)
#pragma unroll 1
                    for (int part = 0; part < (QF32 ? 2 : 1); ++part)
#pragma unroll
                        for (int i = 0; i < D / 16; ++i) {
                            const uint32_t off = ((i / 4) * CU_SUB + (i % 4) * 32) / 16;
                            tc_mma<1>(tmem + 128 * (t % C::SBUFS), q + (part * NSUB * CU_SUB / 16 + off), k + off, id_s, part > 0 || i > 0);
                        }
                    tc_commit(&s_full[t]);
                };
                auto values = [&](int t, uint32_t it, bool keep) {
                    const uint64_t v = vd + (it % NV) * (C::ITEM / 16);
                    const uint32_t tp = tmem + (C::ALIAS ? 128 * t : 128 * C::SBUFS + 64 * t), to = tmem + C::O_COL + D * t;
#pragma unroll(QF32 ? 2 : CU_ROWS / 16)
                    for (int i = 0; i < CU_ROWS / 16; ++i) {
                        const uint64_t b = v + i * (2048 / 16);
                        if constexpr (QF32) {
                            const uint32_t a = tp + 32 * (i / 2) + 8 * (i % 2);
                            tc_mma_ts(to, a, b, id_o, keep || i > 0);
                            tc_mma_ts(to, a + 16, b, id_o, 1);
                        } else {
                            tc_mma_ts(to, tp + 8 * i, b, id_o, keep || i > 0);
                        }
                    }
                    tc_commit(&pv_done[t]);
                };
                auto keys_ready = [&](uint32_t it) { return wait(&k_full[it % NK], it / NK); };
                auto values_ready = [&](uint32_t it) { return wait(&v_full[it % NV], it / NV); };
                for (int e = 0; !*s_abort; ++e) {
                    wait(&r_full[e % CU_RING], e / CU_RING);
                    const RingUnit& R = ring(e);
                    const int state = R.u.state, nt0 = R.nt[0], nt1 = R.nt[1];
                    mbar_arrive(&r_empty[e % CU_RING]);
                    if (state < 0) break;
                    const int nj = max(nt0, nt1);
                    if (nj == 0) continue;
                    auto score_step = [&](int t, int j) {
                        if (j >= (t ? nt1 : nt0)) return;
                        if (j == 0) wait(&q_full[t], t ? nq1++ : nq0++);
                        scores(t, item + j);
                    };
                    auto value_step = [&](int t, int j) {
                        if (j >= (t ? nt1 : nt0)) return;
                        if (!wait(&p_full[t], t ? np1++ : np0++)) return;
                        tc_fence_after();
                        values(t, item + j, j % FOLD != 0);
                    };
                    // the stages of a key (value) tile, once both query tiles' products with it are issued
                    auto keys_done = [&](int j) {
                        tc_commit(&k_empty[(item + j) % NK]);
                        if (j + 1 == nj) tc_commit(q_empty);
                    };
                    if constexpr (C::ALIAS) {
                        // a tile's next scores overwrite its probabilities, so they follow its value product
                        keys_ready(item);
                        score_step(0, 0);
                        score_step(1, 0);
                        keys_done(0);
                        for (int j = 0; j < nj && !*s_abort; ++j) {
                            const bool more = j + 1 < nj;
                            if (more) keys_ready(item + j + 1);
                            values_ready(item + j);
                            value_step(0, j);
                            score_step(0, j + 1);
                            value_step(1, j);
                            score_step(1, j + 1);
                            tc_commit(&v_empty[(item + j) % NV]);
                            if (more) keys_done(j + 1);
                        }
                    } else if (warp == 10) {
                        // scores go out as soon as their buffer was read
                        for (int j = 0; j < nj && !*s_abort; ++j) {
                            keys_ready(item + j);
                            score_step(0, j);
                            score_step(1, j);
                            keys_done(j);
                        }
                    } else {
                        // value products as soon as the probabilities are there
                        for (int j = 0; j < nj && !*s_abort; ++j) {
                            values_ready(item + j);
                            value_step(0, j);
                            value_step(1, j);
                            tc_commit(&v_empty[(item + j) % NV]);
                        }
                    }
                    item += nj;
                }
            }
        } else if (warp >= C::HELPER0) {
            const int ht = tid - 32 * C::HELPER0;  // thread among the helpers
            uint32_t item = 0, cleaned = 0;        // tiles, value tiles cleaned
            for (int e = 0; !stop(); ++e) {
                wait(&r_full[e % CU_RING], e / CU_RING);
                RingUnit& R = ring(e);
                const int state = R.u.state, nj = max(R.nt[0], R.nt[1]), keys = R.u.keys, kt0 = R.t0;
                const int dirty = (R.u.pos0 + 1) / CU_ROWS - R.t0;
                if (state < 0) break;
                if constexpr (SRC == SRC_I8) {
                    // -------------------------------------------------- int8 tiles to fp16, as TMA would lay them out
                    constexpr int CH = D / 16;  // 16-value pieces of a row
                    // (two warps the keys, two the values)
                    const bool is_v = ht >= 64;
                    const int N = is_v ? NV : NK, hh = ht & 63;
                    for (int j = 0; j < nj && !stop(); ++j, ++item) {
                        constexpr uint32_t RR = RAWS > 0 ? RAWS : 1;
                        const uint32_t rs = item % RR, st = item % N;
                        wait((is_v ? rv_full : rk_full) + rs, item / RR);
                        if (item >= N) wait((is_v ? v_empty : k_empty) + st, item / N - 1);
                        const uint4* src = reinterpret_cast<const uint4*>(smem + C::RAW_OFF + ((is_v ? RAWS : 0) + rs) * C::RAW) + hh;
                        uint8_t* dst = smem + C::KV_OFF + ((is_v ? NK : 0) + st) * C::ITEM;
                        // A thread's pieces lie STEP rows apart, a multiple of 8, so their place in the swizzle is
                        // the same. Lanes of the second slice take their halves in the other order: no bank twice.
                        // Not unrolled: beside the softmax loop the instruction cache is what limits (512 queries
                        // after 32 k int8 tokens, fp16 queries: 471 us, 8 pieces at a time 510 us).
                        constexpr int STEP = 64 / CH;
                        const int row = hh / CH, piece = hh % CH, flip = (piece / 4) & 1;
                        uint8_t* slice = dst + (piece / 4) * CU_SUB;
                        uint8_t* d0 = slice + swz_off(row, (piece % 4) * 32 + 16 * flip);
                        uint8_t* d1 = slice + swz_off(row, (piece % 4) * 32 + 16 * (flip ^ 1));
#pragma unroll 1
                        for (int k = 0; k < CU_ROWS; k += STEP) {
                            const uint4 x = src[k * CH];
                            const uint32_t a = (flip ? x.z : x.x) ^ 0x80808080u, b = (flip ? x.w : x.y) ^ 0x80808080u;
                            const uint32_t c = (flip ? x.x : x.z) ^ 0x80808080u, d = (flip ? x.y : x.w) ^ 0x80808080u;
                            *reinterpret_cast<uint4*>(d0 + k * 128) =
                                make_uint4(i8pair_to_h2(a, SEL_B01), i8pair_to_h2(a, SEL_B23), i8pair_to_h2(b, SEL_B01),
                                           i8pair_to_h2(b, SEL_B23));
                            *reinterpret_cast<uint4*>(d1 + k * 128) =
                                make_uint4(i8pair_to_h2(c, SEL_B01), i8pair_to_h2(c, SEL_B23), i8pair_to_h2(d, SEL_B01),
                                           i8pair_to_h2(d, SEL_B23));
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive((is_v ? rv_empty : rk_empty) + rs);
                            mbar_arrive((is_v ? v_full : k_full) + st);
                        }
                    }
                } else {
                    // -------------------------------------------------- values that some row of the unit does not see
                    for (int j = max(0, dirty); j < nj && !stop(); ++j, ++cleaned) {
                        const uint32_t st = (item + j) % NV;
                        wait(&dirty_full[cleaned % CU_CLEAN], cleaned / CU_CLEAN);
                        uint8_t* v = smem + C::KV_OFF + (NK + st) * C::ITEM;
                        const int live_rows = keys - (kt0 + j) * CU_ROWS;  // rows from here on no token sees
                        bool odd = false;
#pragma unroll 8
                        for (int i = ht; i < C::ITEM / 16; i += 32 * C::HELPERS) {
                            uint4* at = reinterpret_cast<uint4*>(v + 16 * i);
                            uint4 x = *at;
                            const __half2 zero = __half2half2(__ushort_as_half(0));
                            // x * 0 is 0 for finite x, NaN otherwise
                            __half2 any = __hfma2(u32_as_h2(x.x), zero, __hmul2(u32_as_h2(x.y), zero));
                            any = __hfma2(u32_as_h2(x.z), zero, __hfma2(u32_as_h2(x.w), zero, any));
                            if ((h2_as_u32(any) & 0x7c007c00u) != 0) {
                                uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                                for (int q = 0; q < 4; ++q) {
                                    if ((w[q] & 0x7c00u) == 0x7c00u) w[q] &= 0xffff0000u;
                                    if ((w[q] & 0x7c000000u) == 0x7c000000u) w[q] &= 0xffffu;
                                }
                                *at = make_uint4(w[0], w[1], w[2], w[3]);
                                odd |= (i * 16 % CU_SUB) / 128 < live_rows;
                            }
                        }
                        if (odd) reinterpret_cast<volatile RingUnit&>(R).odd = 1;
                        fence_proxy_async_smem();
                        __syncwarp();
                        // the last of the four warps hands the tile over
                        if (lane == 0) {
                            __threadfence_block();
                            if (atomicAdd(s_clean + cleaned % CU_CLEAN, 1u) % C::HELPERS == C::HELPERS - 1) {
                                __threadfence_block();
                                mbar_arrive(&v_full[st]);
                            }
                        }
                    }
                    item += nj;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&r_empty[e % CU_RING]);
            }
        }
    }

    if (*s_abort) {
        // a wait gave up: leave this CTA's copies and products in flight two milliseconds to land
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 2000000ull) {}
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 10) tc_dealloc(tmem, 512);
    if (tid == 0 && *s_abort) raise_error(p.error_flag, KVB_DEVERR_TIMEOUT);
}

template <int SRC, bool QF32, int D>
cudaError_t launch(const ChunkParams& p, const CUtensorMap* tq, const CUtensorMap* tk, const CUtensorMap* tv,
                   cudaStream_t stream) {
    using C = CCfg<SRC, QF32, D>;
    static KvbPerDevice<int> configured;
    int done = 0;
    cudaError_t e = configured.get(&done, [](int* v) {
        *v = 1;
        return cudaFuncSetAttribute(chunk_umma_kernel<SRC, QF32, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    int(C::SMEM));
    });
    if (e != cudaSuccess) return e;
    return kvb_launch_pdl(chunk_umma_kernel<SRC, QF32, D>, (unsigned)p.ctas, C::THREADS, C::SMEM, stream, *tq, *tk, *tv, p);
}

template <int SRC, bool QF32>
cudaError_t launch_d(const ChunkParams& p, int D, const CUtensorMap* tq, const CUtensorMap* tk, const CUtensorMap* tv,
                     cudaStream_t stream) {
    return D == 128 ? launch<SRC, QF32, 128>(p, tq, tk, tv, stream) : launch<SRC, QF32, 64>(p, tq, tk, tv, stream);
}

}  // namespace

bool kvb_chunk_umma_supported(int q_type, int kv_type, bool paged, int D, int page, int G) {
    if (D != 64 && D != 128) return false;
    if (G < 1 || G > 64 || (q_type != KVB_F16 && q_type != KVB_F32)) return false;
    if (!paged) return q_type == KVB_F16 && kv_type == KVB_F16;
    if (kv_type != KVB_F16 && kv_type != KVB_I8) return false;
    // a box is a page, or 128 tokens of a larger one
    return page == 8 || page == 16 || page == 32 || page == 64 || page == 128 || page == 256;
}

cudaError_t kvb_launch_chunk_umma(const ChunkParams& p, int q_type, int kv_type, int D, const void* tmap_q,
                                  const void* tmap_k, const void* tmap_v, cudaStream_t stream) {
    const CUtensorMap* tq = static_cast<const CUtensorMap*>(tmap_q);
    const CUtensorMap* tk = static_cast<const CUtensorMap*>(tmap_k);
    const CUtensorMap* tv = static_cast<const CUtensorMap*>(tmap_v);
    if (!p.block_table) return launch_d<SRC_PACKED, false>(p, D, tq, tk, tv, stream);
    if (kv_type == KVB_F16)
        return q_type == KVB_F32 ? launch_d<SRC_F16, true>(p, D, tq, tk, tv, stream)
                                 : launch_d<SRC_F16, false>(p, D, tq, tk, tv, stream);
    return q_type == KVB_F32 ? launch_d<SRC_I8, true>(p, D, tq, tk, tv, stream)
                             : launch_d<SRC_I8, false>(p, D, tq, tk, tv, stream);
}
