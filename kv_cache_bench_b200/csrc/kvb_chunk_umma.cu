// Attention of several new tokens per sequence on B200 tensor cores (tcgen05), with TMA and tensor
// memory; kvb_chunk.cuh has the definition. fp16 or int8 pages, or packed fp16 keys and values; fp32 or
// fp16 queries; head dims 64 and 128.
//
// A query tile is 128 rows, (token, query head of one KV head's group), so that one load of a key tile
// serves the whole group; a unit is two query tiles and 128-key tiles of their keys. Per key tile
//     S[128 rows x 128 keys] = Q K^T      (Q, K in shared memory, K-major)
//     P = exp2(f S - m), l += row sums
//     O[128 rows x D] += P V              (P in tensor memory over S, V in shared memory, MN-major)
// with the running reference m of a row raised only when a score passes it by 2^8 (then O and l are
// scaled in place), so O stays in tensor memory. One persistent CTA per SM:
//   warps 0-3, 4-7  softmax of query tiles 0 and 1, one thread per row (tensor-memory lane): while one
//                   computes its probabilities, the products of the other run. A tile is taken in two
//                   halves of 64 keys, and the products of the first half's probabilities start while
//                   the second's are computed. Probabilities are computed with the reference so far and
//                   the half's maximum beside them; only if that passes it are they computed again.
//   warp 8          TMA producer and unit scheduler: K and V tiles into a ring of stages, Q tiles, and
//                   the units (first blockIdx.x, then one at a time from a counter) through a small ring.
//   warp 9          one thread issues every product, the two query tiles in turn: one tile's products then
//                   run as a block while the other tile's softmax computes. (An issuer per tile let the two
//                   blocks mix, each took twice as long and both groups waited for both: 710 -> 797 us for
//                   a prompt of 8192 tokens.)
//   warp 11         fp16 values: non-finite elements of tiles that some row does not see in full are set
//                   to 0 (0 x inf would not be 0) and, where a row does see them, added at the end.
//   warps 12-15     int8: tiles converted to fp16 (exact), the scales are applied to the scores and to the
//                   probabilities.
// fp32 queries (QF32) keep fp32-level results: q and p are split as fp16(x) + fp16(x - fp16(x)) (about 22
// bits; q prescaled per row by a power of two) and both products run on both halves.
#include <cuda.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "kvb_chunk.cuh"
#include "kvb_tc.cuh"

namespace {

using namespace kvb_dev;

constexpr int CU_ROWS = 128;            // query rows of a tile, keys of a tile
constexpr int CU_SUB = CU_ROWS * 128;   // bytes of [128 rows][128 B], one 128-byte-swizzled slice
constexpr int CU_RING = 4;              // units in flight between the roles
constexpr int CU_POLY = 1, CU_POLY_OF = 4;  // pairs of probabilities on the FMA pipe, of so many
constexpr int CU_CLEAN = 4;             // value tiles on their way to the cleaning warps: at most three are
enum { SRC_F16 = 0, SRC_I8 = 1, SRC_PACKED = 2 };
// The tensor cores add into O with truncation, an error of up to 2^-23 of O per product of 16 keys and in
// one direction. So O is added into an fp32 sum in the workspace (rounded to nearest) and started anew
// every so many key tiles: often for fp32 results, rarely for fp16 ones.
constexpr int CU_FOLD_F32 = KVB_CHUNK_FOLD_F32, CU_FOLD_F16 = KVB_CHUNK_FOLD_F16;
constexpr float CU_TAU = 8.f;    // a row's reference is raised when a score passes it by 2^CU_TAU
constexpr float CU_SHIFT = 6.f;  // probabilities are held times 2^CU_SHIFT: below 2^14, and small ones stay normal

template <int SRC, bool QF32, int D>
struct CCfg {
    static constexpr int NSUB = D / 64;
    static constexpr int ITEM = NSUB * CU_SUB;              // one K or V tile in fp16
    static constexpr int QTILE = NSUB * CU_SUB * (QF32 ? 2 : 1);
    static constexpr int RAW = CU_ROWS * D;                 // one int8 tile
    static constexpr int BUDGET = 227 * 1024 - 1024 - 2048;  // alignment, small arrays
    static constexpr int NR = SRC == SRC_I8 ? (QF32 ? 2 : 3) : 0;
    static constexpr int FIT = (BUDGET - 2 * QTILE - NR * RAW) / ITEM;
    static constexpr int NS = FIT > 6 - NR ? 6 - NR : FIT;  // int8: at most six items in flight (scale ring)
    static constexpr int THREADS = SRC == SRC_I8 ? 512 : 384;
    static constexpr int HELPERS = SRC == SRC_I8 ? 4 : 1;   // converting or cleaning warps
    static constexpr int HELPER0 = SRC == SRC_I8 ? 12 : 11;
    // registers per thread after the split; the launch gives 65536 / THREADS, rounded down to 8
    static constexpr int REGS_LAUNCH = SRC == SRC_I8 ? 128 : 168;
    static constexpr int REGS_SOFT = SRC == SRC_I8 ? 176 : 208;
    static constexpr int REGS_REST = SRC == SRC_I8 ? 80 : 88;
    static_assert(256 * REGS_SOFT + (THREADS - 256) * REGS_REST <= THREADS * REGS_LAUNCH, "register split");
    static constexpr size_t Q_OFF = 0;
    static constexpr size_t KV_OFF = 2 * QTILE;
    static constexpr size_t RAW_OFF = KV_OFF + size_t(NS) * ITEM;
    static constexpr size_t BAR_OFF = RAW_OFF + size_t(NR) * RAW;
    static constexpr int NBARS = 2 * NS + 2 * NR + 13 + CU_CLEAN + 2 * CU_RING;
    static constexpr size_t UNIT_OFF = kvb_align_up(BAR_OFF + 8 * NBARS, 64);
    static constexpr size_t SCALE_OFF = UNIT_OFF + 64 * CU_RING;           // [4 tiles][K, V][16 pages]
    static constexpr size_t VMAX_OFF = SCALE_OFF + (NR ? 4 * 2 * 16 * 4 : 0);  // [4 tiles]
    static constexpr size_t MISC_OFF = kvb_align_up(VMAX_OFF + 16, 16);
    static constexpr size_t SMEM = MISC_OFF + 16 + 1024;
    static_assert(NS >= 2 && SMEM <= 227 * 1024, "shared memory budget");
    static_assert(KV_OFF % 1024 == 0 && RAW_OFF % 1024 == 0, "swizzled tiles need 1024-byte alignment");
};

// A unit as the roles share it.
struct RingUnit {
    ChunkUnit u;
    int t0;         // first key tile
    int nt[2];      // key tiles of the two query tiles
    int odd;        // a seen value was not finite (set by the cleaning warps)
    int bad;        // a block id was refused (set by the producer)
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
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t y;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
    return y;
}

// 2^x of a pair on the FMA pipe: x = n + r with n the nearest integer (the low bits of x + 1.5 * 2^23) and
// r in [-1/2, 1/2], 2^r by its minimax polynomial of degree 4 (fitted to the relative error, 2.6e-6, far
// below the fp16 rounding that follows), n added to its exponent. x is taken as at least -125.
__device__ __forceinline__ void exp2_poly2(uint64_t x, float& a, float& b) {
    unpack2(x, a, b);
    x = pack2(fmaxf(a, -125.f), fmaxf(b, -125.f));
    const uint64_t magic = pack2(12582912.f, 12582912.f), minus = pack2(-12582912.f, -12582912.f);
    const uint64_t n = add2(x, magic);
    const uint64_t r = fma2(add2(n, minus), pack2(-1.f, -1.f), x);
    uint64_t y = fma2(r, pack2(0.009570102207362652f, 0.009570102207362652f), pack2(0.05591785907745361f, 0.05591785907745361f));
    y = fma2(y, r, pack2(0.240247443318367f, 0.240247443318367f));
    y = fma2(y, r, pack2(0.6931217908859253f, 0.6931217908859253f));
    y = fma2(y, r, pack2(0.9999992847442627f, 0.9999992847442627f));
    float na, nb;
    unpack2(n, na, nb);
    unpack2(y, a, b);
    a = __uint_as_float(__float_as_uint(a) + (__float_as_uint(na) << 23));
    b = __uint_as_float(__float_as_uint(b) + (__float_as_uint(nb) << 23));
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
    constexpr int NSUB = C::NSUB, NS = C::NS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = smem_u32(smem);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);  // [NS] K or V tile ready for the products
    uint64_t* empty = full + NS;         // [NS] its products are done
    uint64_t* raw_full = empty + NS;     // [NR] int8 tile loaded
    uint64_t* raw_empty = raw_full + C::NR;
    uint64_t* q_full = raw_empty + C::NR;  // [2] query tile in shared memory
    uint64_t* q_empty = q_full + 2;      // both query tiles' score products are done
    uint64_t* s_full = q_empty + 1;      // [2] scores ready, and every product before them done
    uint64_t* p_full = s_full + 2;       // [2][2 halves] probabilities written, O scaled
    uint64_t* half_done = p_full + 4;    // [2] the products of the first half done
    uint64_t* o_full = half_done + 2;    // [2] the unit's O complete
    uint64_t* dirty_full = o_full + 2;   // [CU_CLEAN] a value tile loaded that passes the cleaning warps first
    uint64_t* r_full = dirty_full + CU_CLEAN;  // [CU_RING] unit published
    uint64_t* r_empty = r_full + CU_RING;
    auto ring = [&](int e) -> RingUnit& { return *reinterpret_cast<RingUnit*>(smem + C::UNIT_OFF + 64 * (e % CU_RING)); };
    float* s_scale = reinterpret_cast<float*>(smem + C::SCALE_OFF);
    float* s_vmax = reinterpret_cast<float*>(smem + C::VMAX_OFF);
    volatile int* s_abort = reinterpret_cast<volatile int*>(smem + C::MISC_OFF);
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + C::MISC_OFF + 8);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (warp == 0) {
        for (int i = lane; i < C::NBARS; i += 32) {
            uint64_t* b = full + i;
            uint32_t n = 1;
            if (b < empty) n = SRC == SRC_I8 ? C::HELPERS : 1;
            else if (b >= raw_empty && b < q_full) n = C::HELPERS;
            else if (b >= q_full && b < q_empty) n = QF32 ? 4 : 1;
            else if (b >= p_full && b < half_done) n = 4;
            else if (b >= r_empty) n = 1 + 8 + C::HELPERS;  // product issuer, softmax warps, helpers
            mbar_init(b, n);
        }
        if (lane == 0) *s_abort = 0;
        fence_mbarrier_init();
    }
    if (warp == 9) {
        tc_alloc(s_tmem, 512);
        tc_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;  // columns: S/P of tile t at 128 t, O of tile t at 256 + D t
    pdl_wait();
    pdl_trigger();

    // False once a wait has given up (here, or elsewhere in the CTA where this one would block).
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (mbar_try_wait(bar, parity & 1)) return true;
        if (!*s_abort && mbar_wait_bounded(bar, parity & 1, s_abort)) return true;
        *s_abort = 1;
        return false;
    };
    auto stop = [&]() { return __any_sync(0xffffffffu, *s_abort) != 0; };  // the same answer in a whole warp

    if (warp < 8) {
        // ---------------------------------------------------------------- softmax, one thread per query row
        reg_alloc<C::REGS_SOFT>();
        const int t = warp >> 2;
        const int r = tid & 127;  // row of the tile
        const uint32_t lanes = uint32_t(warp & 3) << 21;  // this warp's quarter of the tensor-memory lanes
        const uint32_t ts = tmem + lanes + 128 * t, to = tmem + lanes + 256 + D * t;
        const int tok = r / p.G, head = r % p.G;
        const int lp = SRC == SRC_I8 ? __ffs(p.page) - 1 : 0;
        uint32_t ns = 0, no = 0;  // score tiles and units that this group has taken
        uint32_t tiles = 0;       // key tiles of the CTA so far (int8 scale ring)
        constexpr int FOLD = QF32 ? CU_FOLD_F32 : CU_FOLD_F16;
        float4* fold = reinterpret_cast<float4*>(p.fold) + (size_t)(2 * blockIdx.x + t) * (D / 4) * 128 + r;
        for (int e = 0;; ++e) {
            wait(&r_full[e % CU_RING], e / CU_RING);
            const RingUnit& R = ring(e);
            const ChunkUnit u = R.u;
            const int nt = R.nt[t], nall = max(R.nt[0], R.nt[1]), kt0 = R.t0;
            if (u.state < 0 || stop()) break;
            auto leave = [&]() {
                __syncwarp();
                if (lane == 0) mbar_arrive(&r_empty[e % CU_RING]);
            };
            if (u.state == 2) {
                if (t == 0) chunk_refuse<QT, D>(p, u, r, 128);
                leave();
                continue;
            }
            const int tt = t * p.tile_tokens;              // first token of the tile in the unit
            const int cnt = min(u.n - tt, p.tile_tokens);  // its tokens
            if (cnt <= 0) {
                tiles += nall;
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
                    // this row's query, split; the tile's previous scores are done (this group waited for them)
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
                    x = amax > 0.f && x < 128 ? max(x, -100) : 0;
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
            float l = 0.f;
            float vexp = 0.f;       // int8: 2^-e, probabilities times the value scales times this; 0: not set
            float older = 1.f;      // what the folded sum has to be scaled by
            int folds = 0;
            // O (complete up to here) and the folded sum times `scale`
            auto rescale = [&](float scale) {
                older *= scale;
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    uint32_t o[32];
                    tc_ld32(to + c, o);
                    tc_wait_ld();
                    pin<32>(o);
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * scale);
                    tc_st32(to + c, o);
                }
            };
            for (int j = 0; j < nt; ++j) {
                if (__any_sync(0xffffffffu, !wait(&s_full[t], ns))) break;
                tc_fence_after();
                const int k0 = (kt0 + j) * CU_ROWS;
                const bool masked = k0 + CU_ROWS > all_see;
                const float* scales = s_scale + ((tiles + j) & 3) * 32;
                if (j > 0 && j % FOLD == 0) {
                    // the products of the tiles before are done, the next one starts O anew
                    const bool plain = __all_sync(0xffffffffu, older == 1.f);
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        uint32_t o[32];
                        tc_ld32(to + c, o);
                        tc_wait_ld();
                        pin<32>(o);
                        float4* at = fold + (c / 4) * 128;
#pragma unroll
                        for (int i = 0; i < 8; ++i, at += 128) {
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
                    const float vm = s_vmax[(tiles + j) & 3];  // the tile's largest finite value scale
                    if (vexp == 0.f || vm * vexp > 2.f) {      // (the same in every row)
                        const int x = min(max(int(__float_as_uint(vm) >> 23) - 127, -100), 125);
                        const float ve = __uint_as_float(uint32_t(126 - x) << 23);  // vm * ve in [0.5, 1)
                        if (vexp != 0.f) rescale(ve / vexp);
                        vexp = ve;
                    }
                }
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {
                    uint32_t s[64];
                    tc_ld32(ts + 64 * half, s);
                    tc_ld32(ts + 64 * half + 32, s + 32);
                    tc_wait_ld();
                    pin<64>(s);
                    const int kh = k0 + 64 * half;
                    if constexpr (SRC == SRC_I8) {
#pragma unroll
                        for (int c = 0; c < 64; c += 8) {
                            const float ks = scales[(64 * half + c) >> lp];  // (pages of 128 tokens or more: one)
#pragma unroll
                            for (int i = 0; i < 8; ++i) s[c + i] = __float_as_uint(__uint_as_float(s[c + i]) * ks);
                        }
                    }
                    if (masked) {
                        const int lim = limit - kh;
#pragma unroll
                        for (int c = 0; c < 64; ++c)
                            if (c >= lim) s[c] = 0xff800000u;  // -inf
                    }
                    uint32_t pr[QF32 ? 64 : 32];
                    float sum, mt;
                    auto probabilities = [&](float base) {
                        const uint64_t f2 = pack2(f, f), b2 = pack2(base, base);
                        uint64_t l0 = 0, l1 = 0;
                        float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
                        for (int i = 0; i < 64; i += 2) {
                            const float s0 = __uint_as_float(s[i]), s1 = __uint_as_float(s[i + 1]);
                            if (i & 2) m1 = max3_nan(m1, s0, s1);
                            else m0 = max3_nan(m0, s0, s1);
                            const uint64_t x = fma2(pack2(s0, s1), f2, b2);
                            float a, b;
                            if (!QF32 && (i / 2) % CU_POLY_OF < CU_POLY) {
                                exp2_poly2(x, a, b);
                            } else {
                                unpack2(x, a, b);
                                a = ex2(a);
                                b = ex2(b);
                            }
                            if (i & 2) l1 = add2(l1, pack2(a, b));
                            else l0 = add2(l0, pack2(a, b));
                            if constexpr (SRC == SRC_I8) {
                                const float vs = scales[16 + ((64 * half + i) >> lp)] * vexp;
                                a *= vs;
                                b *= vs;
                                if (masked) {  // the scale of a page that this row does not see may be anything
                                    if (kh + i >= limit) a = 0.f;
                                    if (kh + i + 1 >= limit) b = 0.f;
                                }
                            }
                            if constexpr (QF32) split_hi_lo(a, b, pr[32 * (i / 32) + i % 32 / 2], pr[32 * (i / 32) + 16 + i % 32 / 2]);
                            else pr[i / 2] = h2_as_u32(__floats2half2_rn(a, b));
                        }
                        float a, b;
                        unpack2(add2(l0, l1), a, b);
                        sum = a + b;
                        mt = fmaxf_nan(m0, m1);
                    };
                    bool move = j == 0 && half == 0;
                    if (!move) {
                        probabilities(ref == -INFINITY ? 0.f : -ref);
                        move = mt * f - CU_SHIFT > ref + CU_TAU;
                    } else {
                        float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
                        for (int i = 0; i < 64; i += 4) {
                            m0 = max3_nan(m0, __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
                            m1 = max3_nan(m1, __uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
                        }
                        mt = fmaxf_nan(m0, m1);
                    }
                    if (__any_sync(0xffffffffu, move)) {
                        // a new reference where a score passed the old one: O, l and these probabilities follow
                        float scale = 1.f;
                        const float top = mt * f - CU_SHIFT;
                        if (top > ref) {
                            scale = ref == -INFINITY ? 0.f : ex2(ref - top);
                            ref = top;
                            l *= scale;
                        }
                        if (j > 0 || half) {
                            if (half) wait(&half_done[t], ns);
                            tc_fence_after();
                            rescale(scale);
                        }
                        probabilities(ref == -INFINITY ? 0.f : -ref);
                    }
                    // a NaN or +inf score makes the whole row NaN
                    l += mt < INFINITY ? sum : __int_as_float(0x7fc00000);
                    if constexpr (QF32) {  // hi, lo of 32 keys: 16 columns each
                        tc_st32(ts + 64 * half, pr);
                        tc_st32(ts + 64 * half + 32, pr + 32);
                    } else {
                        tc_st32(ts + 32 * half, pr);
                    }
                    tc_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_full[2 * t + half]);
                }
                ++ns;
            }
            tiles += nall;
            if (nt > 0) {
                wait(&o_full[t], no);
                ++no;
                tc_fence_after();
            }
            if (stop()) break;
            const volatile RingUnit& V = R;
            const bool bad = V.bad != 0, odd = V.odd != 0;
            if (bad && r == 0) raise_error(p.error_flag, KVB_DEVERR_BLOCK);
            float inv = bad ? __int_as_float(0x7fc00000) : p.splits > 1 && l == 0.f ? 0.f : 1.f / l;
            const size_t row = (size_t)qrow * p.H + h;
            const size_t at = (size_t)u.split * p.T * p.H + row;
            if (p.splits > 1 && live) p.part_ml[at] = make_float2(ref, bad ? inv : l);
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
                    const int first = max(kt0, all_see / CU_ROWS) * CU_ROWS;
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
                } else if (QF32 || p.splits > 1) {
                    uint4* out = reinterpret_cast<uint4*>(p.splits > 1 ? p.part_o + at * D + c
                                                                       : static_cast<float*>(p.out) + row * D + c);
#pragma unroll
                    for (int i = 0; i < 8; ++i) out[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                } else {
                    uint4* out = reinterpret_cast<uint4*>(static_cast<__half*>(p.out) + row * D + c);
                    auto h2 = [&](int i) {
                        return h2_as_u32(__floats2half2_rn(__uint_as_float(o[i]), __uint_as_float(o[i + 1])));
                    };
#pragma unroll
                    for (int i = 0; i < 4; ++i) out[i] = make_uint4(h2(8 * i), h2(8 * i + 2), h2(8 * i + 4), h2(8 * i + 6));
                }
            }
            tc_fence_before();
            leave();
        }
    } else {
        reg_dealloc<C::REGS_REST>();
        if (warp == 8) {
            // ------------------------------------------------------------ producer and scheduler
            const uint64_t policy = l2_evict_first_policy();
            uint32_t item = 0, tiles = 0, units = 0;
            uint32_t qn = 0;  // units whose queries were loaded
            uint32_t dirty_n = 0;  // value tiles sent to the cleaning warps
            long long idx = blockIdx.x;
            auto next = [&]() {
                long long i = p.units;
                if (p.next_unit && lane == 0) i = (long long)gridDim.x + atomicAdd(p.next_unit, 1u);
                return p.next_unit ? __shfl_sync(0xffffffffu, i, 0) : i;
            };
            auto publish = [&](const ChunkUnit& u, int2 range, int nt0, int nt1) {
                if (units >= CU_RING) wait(&r_empty[units % CU_RING], units / CU_RING - 1);
                __syncwarp();
                if (lane == 0) {
                    RingUnit& R = ring(units);
                    R.u = u;
                    R.t0 = range.x;
                    R.nt[0] = nt0;
                    R.nt[1] = nt1;
                    R.odd = R.bad = 0;
                    mbar_arrive(&r_full[units % CU_RING]);
                }
                ++units;
            };
            for (; idx < p.units && !stop(); idx = next()) {
                const ChunkUnit u = chunk_unit(p, idx);
                if (u.state == 1) continue;
                if (u.state == 2) {
                    publish(u, make_int2(0, 0), 0, 0);
                    continue;
                }
                const int2 range = chunk_split_tiles(p, u, CU_ROWS);
                const int n1 = u.n - p.tile_tokens;  // tokens of tile 1
                const int keys0 = u.pos0 + min(u.n, p.tile_tokens);
                const int nt0 = max(0, min(range.y, (keys0 + CU_ROWS - 1) / CU_ROWS) - range.x);
                const int nt1 = n1 > 0 ? range.y - range.x : 0;
                const int dirty = (u.pos0 + 1) / CU_ROWS - range.x;  // values from this tile on pass the cleaning warps
                const int e = units;
                publish(u, range, nt0, nt1);
                const int nj = max(nt0, nt1);
                if (nj == 0) continue;
                const int bt = SRC == SRC_PACKED ? CU_ROWS : min(p.page, CU_ROWS);  // keys of a box
                const int nbox = CU_ROWS / bt;
                const int* table = p.block_table + (SRC == SRC_PACKED ? 0 : (size_t)u.b * p.max_blocks);
                // the block id (int8: and scales) of this lane's box of a tile, one tile ahead
                int id = -1, nid = -1;
                auto fetch = [&](int j) {
                    const int k = (range.x + j) * CU_ROWS + lane * bt;
                    return SRC != SRC_PACKED && j < nj && lane < nbox && k < u.keys ? __ldg(table + k / p.page) : -1;
                };
                nid = fetch(0);
                for (int j = 0; j < nj && !stop(); ++j) {
                    id = nid;
                    nid = fetch(j + 1);
                    const int k = (range.x + j) * CU_ROWS + lane * bt;
                    const bool wanted = SRC != SRC_PACKED && lane < nbox && k < u.keys;
                    const bool ok = wanted && id >= 0 && id < p.num_blocks;
                    if (__any_sync(0xffffffffu, wanted && !ok) && lane == 0)
                        reinterpret_cast<volatile RingUnit&>(ring(e)).bad = 1;
                    const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, ok));
                    if constexpr (SRC == SRC_I8) {
                        float ks = 0.f, vs = 0.f;
                        if (ok) {
                            ks = __ldg(p.k_scale + (long long)id * p.Hkv + u.kvh);
                            vs = __ldg(p.v_scale + (long long)id * p.Hkv + u.kvh);
                        }
                        // the ring's slot: its readers are done, since the item six before this one is
                        if (item >= C::NR) wait(&raw_empty[item % C::NR], item / C::NR - 1);
                        const float vm = warp_max(vs <= 3.402823466e38f ? vs : 0.f);
                        if (lane < 16) {
                            s_scale[(tiles & 3) * 32 + lane] = ks;
                            s_scale[(tiles & 3) * 32 + 16 + lane] = vs;
                        }
                        if (lane == 0) s_vmax[tiles & 3] = vm;
                    }
#pragma unroll
                    for (int which = 0; which < 2; ++which) {  // K, then V
                        if constexpr (SRC == SRC_I8) {
                            const uint32_t st = item % C::NR;
                            if (item >= C::NR) wait(&raw_empty[st], item / C::NR - 1);
                            __syncwarp();
                            const uint32_t bytes = uint32_t(bt) * D;
                            if (lane == 0) {
                                if (boxes && !*s_abort) mbar_arrive_expect_tx(&raw_full[st], boxes * bytes);
                                else mbar_arrive(&raw_full[st]);
                            }
                            __syncwarp();
                            if (ok && !*s_abort) {
                                const int8_t* src = static_cast<const int8_t*>(which ? p.v : p.k) +
                                                    (((long long)id * p.Hkv + u.kvh) * p.page + k % p.page) * D;
                                bulk_load(smem + C::RAW_OFF + st * C::RAW + lane * bytes, src, bytes, &raw_full[st]);
                            }
                        } else {
                            const uint32_t st = item % NS;
                            if (item >= NS) wait(&empty[st], item / NS - 1);
                            __syncwarp();
                            uint8_t* dst = smem + C::KV_OFF + st * C::ITEM;
                            const CUtensorMap* map = which ? &tmv : &tmk;
                            uint64_t* done = &full[st];
                            if (which && j >= dirty) done = &dirty_full[dirty_n++ % CU_CLEAN];
                            if constexpr (SRC == SRC_PACKED) {
                                if (lane == 0) {
                                    if (*s_abort) {
                                        mbar_arrive(done);
                                    } else {
                                        mbar_arrive_expect_tx(done, C::ITEM);
#pragma unroll
                                        for (int i = 0; i < NSUB; ++i)
                                            tma_load_3d(dst + i * CU_SUB, map, done, 64 * i, u.kvh,
                                                        u.kv0 + (range.x + j) * CU_ROWS);
                                    }
                                }
                            } else {
                                if (lane == 0) {
                                    if (boxes && !*s_abort) mbar_arrive_expect_tx(done, boxes * bt * 128 * NSUB);
                                    else mbar_arrive(done);
                                }
                                __syncwarp();
                                if (ok && !*s_abort) {
                                    const int y = (id * p.Hkv + u.kvh) * p.page + k % p.page;
#pragma unroll
                                    for (int i = 0; i < NSUB; ++i)
                                        tma_load_2d(dst + i * CU_SUB + lane * bt * 128, map, done, 64 * i, y, policy);
                                }
                            }
                        }
                        ++item;
                        if (!QF32 && j == 0 && which == 0) {
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
                                    for (int i = 0; i < NSUB; ++i)
                                        tma_load_3d(smem + C::Q_OFF + t * C::QTILE + i * CU_SUB, &tmq, &q_full[t], 64 * i,
                                                    u.kvh * p.G, u.row0 + t * p.tile_tokens);
                                }
                            }
                            __syncwarp();
                        }
                    }
                    ++tiles;
                }
            }
            ChunkUnit end{};
            end.state = -1;
            publish(end, make_int2(0, 0), 0, 0);
        } else if (warp == 9) {
            // ------------------------------------------------------------ products
            if (tc_elect()) {
                constexpr uint32_t id_s = instr_desc(1, 0, 0, 0, 0, 128, 128);
                constexpr uint32_t id_o = instr_desc(1, 0, 0, 0, 1, D, 128);
                constexpr int FOLD = QF32 ? CU_FOLD_F32 : CU_FOLD_F16;
                // descriptors of the first stage; a byte offset of o adds o / 16
                const uint64_t kd = smem_desc(sbase + uint32_t(C::KV_OFF), 16, 1024);
                const uint64_t vd = smem_desc(sbase + uint32_t(C::KV_OFF), CU_SUB, 1024);
                const uint64_t qd = smem_desc(sbase + uint32_t(C::Q_OFF), 16, 1024);
                uint32_t item = 0, nq0 = 0, nq1 = 0, np0 = 0, np1 = 0;
                auto scores = [&](int t, uint32_t it) {
                    const uint64_t k = kd + (it % NS) * (C::ITEM / 16), q = qd + t * (C::QTILE / 16);
#pragma unroll
                    for (int part = 0; part < (QF32 ? 2 : 1); ++part)
#pragma unroll
                        for (int i = 0; i < D / 16; ++i) {
                            const uint32_t off = ((i / 4) * CU_SUB + (i % 4) * 32) / 16;
                            tc_mma<1>(tmem + 128 * t, q + (part * NSUB * CU_SUB / 16 + off), k + off, id_s, part > 0 || i > 0);
                        }
                    tc_commit(&s_full[t]);
                };
                auto values = [&](int t, uint32_t it, int half, bool keep) {
                    const uint64_t v = vd + (it % NS) * (C::ITEM / 16) + half * (64 * 128 / 16);
                    const uint32_t ts = tmem + 128 * t + (QF32 ? 64 : 32) * half, to = tmem + 256 + D * t;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint64_t b = v + i * (2048 / 16);
                        if constexpr (QF32) {
                            const uint32_t a = ts + 32 * (i / 2) + 8 * (i % 2);
                            tc_mma_ts(to, a, b, id_o, keep || i > 0);
                            tc_mma_ts(to, a + 16, b, id_o, 1);
                        } else {
                            tc_mma_ts(to, ts + 8 * i, b, id_o, keep || i > 0);
                        }
                    }
                };
                auto ready = [&](uint32_t it) { return wait(&full[it % NS], it / NS); };
                for (int e = 0; !*s_abort; ++e) {
                    wait(&r_full[e % CU_RING], e / CU_RING);
                    const RingUnit& R = ring(e);
                    const int state = R.u.state, nt0 = R.nt[0], nt1 = R.nt[1];
                    mbar_arrive(&r_empty[e % CU_RING]);
                    if (state < 0) break;
                    const int nj = max(nt0, nt1);
                    if (nj == 0) continue;
                    // K of key tile j is item `item` + 2 j, its V the next one
                    ready(item);
                    if (nt0 > 0) {
                        wait(&q_full[0], nq0++);
                        tc_fence_after();
                        scores(0, item);
                    }
                    if (nt1 > 0) {
                        wait(&q_full[1], nq1++);
                        tc_fence_after();
                        scores(1, item);
                    }
                    tc_commit(&empty[item % NS]);
                    if (nj == 1) tc_commit(q_empty);
                    for (int j = 0; j < nj && !*s_abort; ++j) {
                        const uint32_t iv = item + 1, ik = item + 2;
                        bool have_k = false;
                        ready(iv);
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            const int nt = t ? nt1 : nt0;
                            if (j >= nt) continue;
                            uint32_t& np = t ? np1 : np0;
                            if (!wait(&p_full[2 * t], np)) break;
                            tc_fence_after();
                            values(t, iv, 0, j % FOLD != 0);
                            tc_commit(&half_done[t]);
                            if (j + 1 < nt && !have_k) have_k = ready(ik);  // while the second half is computed
                            if (!wait(&p_full[2 * t + 1], np)) break;
                            tc_fence_after();
                            values(t, iv, 1, true);
                            ++np;
                            if (j + 1 < nt) {
                                scores(t, ik);
                            } else {
                                tc_commit(&o_full[t]);
                            }
                        }
                        tc_commit(&empty[iv % NS]);
                        if (j + 1 < nj) tc_commit(&empty[ik % NS]);
                        if (j + 2 == nj) tc_commit(q_empty);
                        item += 2;
                    }
                }
            }
        } else if (warp >= C::HELPER0) {
            const int ht = tid - 32 * C::HELPER0;  // thread among the helpers
            uint32_t item = 0, cleaned = 0;  // cleaned: value tiles taken
            for (int e = 0; !stop(); ++e) {
                wait(&r_full[e % CU_RING], e / CU_RING);
                RingUnit& R = ring(e);
                const int state = R.u.state, nj = max(R.nt[0], R.nt[1]), keys = R.u.keys, kt0 = R.t0;
                const int dirty = (R.u.pos0 + 1) / CU_ROWS - R.t0;
                if (state < 0) break;
                if constexpr (SRC == SRC_I8) {
                    // -------------------------------------------------- int8 tiles to fp16, as TMA would lay them out
                    constexpr int CH = D / 16;  // 16-value pieces of a row
                    for (int k = 0; k < 2 * nj && !stop(); ++k, ++item) {
                        const uint32_t rs = item % C::NR, st = item % NS;
                        wait(&raw_full[rs], item / C::NR);
                        if (item >= NS) wait(&empty[st], item / NS - 1);
                        const uint4* src = reinterpret_cast<const uint4*>(smem + C::RAW_OFF + rs * C::RAW);
                        uint8_t* dst = smem + C::KV_OFF + st * C::ITEM;
#pragma unroll 4
                        for (int i = ht; i < CU_ROWS * CH; i += 32 * C::HELPERS) {
                            const uint4 x = src[i];
                            const int row = i / CH, c = i % CH;
                            const uint32_t w[4] = {x.x ^ 0x80808080u, x.y ^ 0x80808080u, x.z ^ 0x80808080u, x.w ^ 0x80808080u};
                            uint4 y[2];
                            y[0] = make_uint4(i8pair_to_h2(w[0], SEL_B01), i8pair_to_h2(w[0], SEL_B23),
                                              i8pair_to_h2(w[1], SEL_B01), i8pair_to_h2(w[1], SEL_B23));
                            y[1] = make_uint4(i8pair_to_h2(w[2], SEL_B01), i8pair_to_h2(w[2], SEL_B23),
                                              i8pair_to_h2(w[3], SEL_B01), i8pair_to_h2(w[3], SEL_B23));
                            // lanes of the second slice store their halves in the other order: no bank twice
                            uint8_t* slice = dst + (c / 4) * CU_SUB;
                            const int flip = (c / 4) & 1;
                            const uint32_t o0 = swz_off(row, (c % 4) * 32), o1 = swz_off(row, (c % 4) * 32 + 16);
                            *reinterpret_cast<uint4*>(slice + (flip ? o1 : o0)) = flip ? y[1] : y[0];
                            *reinterpret_cast<uint4*>(slice + (flip ? o0 : o1)) = flip ? y[0] : y[1];
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive(&raw_empty[rs]);
                            mbar_arrive(&full[st]);
                        }
                    }
                } else {
                    // -------------------------------------------------- values that some row of the unit does not see
                    // (the two warps take them in turn)
                    for (int j = max(0, dirty); j < nj && !stop(); ++j, ++cleaned) {
                        if (int(cleaned % C::HELPERS) != ht >> 5) continue;
                        const uint32_t it = item + 2 * j + 1;
                        wait(&dirty_full[cleaned % CU_CLEAN], cleaned / CU_CLEAN);
                        uint8_t* v = smem + C::KV_OFF + (it % NS) * C::ITEM;
                        const int live_rows = keys - (kt0 + j) * CU_ROWS;  // rows from here on no token sees
                        bool odd = false;
#pragma unroll 8
                        for (int i = lane; i < C::ITEM / 16; i += 32) {
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
                        if (lane == 0) mbar_arrive(&full[it % NS]);
                    }
                    item += 2 * nj;
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
    if (warp == 9) tc_dealloc(tmem, 512);
    if (tid == 0 && *s_abort) raise_error(p.error_flag, KVB_DEVERR_TIMEOUT);
}

template <int SRC, bool QF32, int D>
cudaError_t launch(const ChunkParams& p, const CUtensorMap* tq, const CUtensorMap* tk, const CUtensorMap* tv,
                   int num_sms, cudaStream_t stream) {
    using C = CCfg<SRC, QF32, D>;
    static KvbPerDevice<int> configured;
    int done = 0;
    cudaError_t e = configured.get(&done, [](int* v) {
        *v = 1;
        return cudaFuncSetAttribute(chunk_umma_kernel<SRC, QF32, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    int(C::SMEM));
    });
    if (e != cudaSuccess) return e;
    const long long grid = std::min<long long>(p.units, num_sms);
    if (p.next_unit) {
        e = cudaMemsetAsync(p.next_unit, 0, sizeof(unsigned), stream);
        if (e != cudaSuccess) return e;
    }
    return kvb_launch_pdl(chunk_umma_kernel<SRC, QF32, D>, (unsigned)grid, C::THREADS, C::SMEM, stream, *tq, *tk, *tv, p);
}

template <int SRC, bool QF32>
cudaError_t launch_d(const ChunkParams& p, int D, const CUtensorMap* tq, const CUtensorMap* tk, const CUtensorMap* tv,
                     int num_sms, cudaStream_t stream) {
    return D == 128 ? launch<SRC, QF32, 128>(p, tq, tk, tv, num_sms, stream)
                    : launch<SRC, QF32, 64>(p, tq, tk, tv, num_sms, stream);
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
                                  const void* tmap_k, const void* tmap_v, int num_sms, cudaStream_t stream) {
    const CUtensorMap* tq = static_cast<const CUtensorMap*>(tmap_q);
    const CUtensorMap* tk = static_cast<const CUtensorMap*>(tmap_k);
    const CUtensorMap* tv = static_cast<const CUtensorMap*>(tmap_v);
    if (!p.block_table) return launch_d<SRC_PACKED, false>(p, D, tq, tk, tv, num_sms, stream);
    if (kv_type == KVB_F16)
        return q_type == KVB_F32 ? launch_d<SRC_F16, true>(p, D, tq, tk, tv, num_sms, stream)
                                 : launch_d<SRC_F16, false>(p, D, tq, tk, tv, num_sms, stream);
    return q_type == KVB_F32 ? launch_d<SRC_I8, true>(p, D, tq, tk, tv, num_sms, stream)
                             : launch_d<SRC_I8, false>(p, D, tq, tk, tv, num_sms, stream);
}
