// Attention of several new tokens per sequence on CUDA cores (fp32 caches, and every shape and page
// size that the tcgen05 kernel does not take), and the merge of split keys. kvb_chunk.cuh has the
// definition; the reference's decode kernel (src/kernels.metal:43-147) is the case of one new token.
#include <cuda_fp16.h>

#include <algorithm>

#include "kvb_chunk.cuh"

namespace {

using namespace kvb_dev;

constexpr int SM_THREADS = 128;
constexpr int SM_ROWS = KVB_SIMT_ROWS;  // query rows of a tile: (token, head of the group)
constexpr int SM_KEYS = 32;             // keys of a tile

// One unit per CTA: a tile of 64 query rows against tiles of 32 keys, everything in fp32. Thread (rg,
// cg), 16 x 8, holds scores of rows rg + 16 i and keys cg + 8 j (4 x 4) and the outputs of the same
// rows, dims 4 (cg + 8 c) .. + 3. Rows of the shared tiles are padded by four floats, so that the rows
// a warp reads together lie in different banks. 16 shared-memory loads of 16 bytes feed 256 FMAs of a
// thread, with a wavefront each, half of the FMAs' time. Bound by latency: a tile's table read, row pointers,
// loads and three barriers follow one another, with eight warps on an SM and nothing of the next tile on its way
// (2 x 61 tokens on 451, 32 heads of 128: 58 us, 13 at the FMA rate; a prompt of 1024: 359, 125).
template <int D>
struct SimtCfg {
    static constexpr int LD = D + 4;
    static constexpr int LP = SM_KEYS + 4;
    static constexpr size_t Q_OFF = 0;
    static constexpr size_t K_OFF = Q_OFF + sizeof(float) * SM_ROWS * LD;
    static constexpr size_t V_OFF = K_OFF + sizeof(float) * SM_KEYS * LD;
    static constexpr size_t P_OFF = V_OFF + sizeof(float) * SM_KEYS * LD;
    static constexpr size_t SMEM = P_OFF + sizeof(float) * SM_ROWS * LP;
};

template <typename T>
__device__ __forceinline__ float4 load_row4(const T* s, float scale) {
    if constexpr (sizeof(T) == 4) {
        return *reinterpret_cast<const float4*>(s);
    } else if constexpr (sizeof(T) == 2) {
        const uint2 r = *reinterpret_cast<const uint2*>(s);
        const float2 a = __half22float2(u32_as_h2(r.x)), b = __half22float2(u32_as_h2(r.y));
        return make_float4(a.x, a.y, b.x, b.y);
    } else {
        const char4 c = *reinterpret_cast<const char4*>(s);
        return make_float4(c.x * scale, c.y * scale, c.z * scale, c.w * scale);
    }
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }

template <typename QT, typename KT, int D>
__global__ void __launch_bounds__(SM_THREADS) chunk_simt_kernel(const __grid_constant__ ChunkParams p) {
    using C = SimtCfg<D>;
    constexpr int D4 = D / 4, OC = D4 / 8;  // float4 pieces of a row; of a thread's outputs
    extern __shared__ __align__(16) uint8_t smem[];
    float* sq = reinterpret_cast<float*>(smem + C::Q_OFF);
    float* sk = reinterpret_cast<float*>(smem + C::K_OFF);
    float* sv = reinterpret_cast<float*>(smem + C::V_OFF);
    float* sp = reinterpret_cast<float*>(smem + C::P_OFF);
    __shared__ const KT* s_rows[2][SM_KEYS];
    __shared__ float s_scale[2][SM_KEYS];
    __shared__ int s_bad, s_odd;  // first position whose block id was refused; a masked value was not finite
    const int tid = threadIdx.x, rg = tid >> 3, cg = tid & 7;
    pdl_wait();
    pdl_trigger();
    const ChunkUnit u = chunk_unit(p, blockIdx.x);
    if (u.state == 1) return;
    if (u.state == 2) {
        chunk_refuse<QT, D>(p, u, tid, SM_THREADS);
        return;
    }
    const int h0 = u.kvh * p.G;
    const int rows = u.n * p.G;  // <= SM_ROWS
    if (tid == 0) {
        s_bad = 0x7fffffff;
        s_odd = 0;
    }
    for (int i = tid; i < SM_ROWS * D4; i += SM_THREADS) {
        const int r = i / D4, c = i % D4;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < rows)
            x = load_row4(static_cast<const QT*>(p.q) + (long long)(u.row0 + r / p.G) * p.q_stride +
                              (long long)(h0 + r % p.G) * D + 4 * c, 1.f);
        *reinterpret_cast<float4*>(sq + r * C::LD + 4 * c) = x;
    }
    int limit[4];  // keys that this thread's rows see
#pragma unroll
    for (int i = 0; i < 4; ++i) limit[i] = u.pos0 + min(rg + 16 * i, rows - 1) / p.G + 1;
    float m[4], l[4];
    float4 o[4][OC];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < OC; ++c) o[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const int2 tiles = chunk_split_tiles(p, u, SM_KEYS);
    const int seen_by_all = u.pos0 + 1;  // keys that every row of the unit sees
    for (int t = tiles.x; t < tiles.y; ++t) {
        const int k0 = t * SM_KEYS;
        __syncthreads();  // the tiles of the round before were read
        if (tid < 2 * SM_KEYS) {
            const int j = tid & (SM_KEYS - 1), which = tid / SM_KEYS;
            const KT* row = nullptr;
            float sc = 0.f;
            if (k0 + j < u.keys) {
                row = which ? chunk_row<KT>(p, u, p.v, p.v_stride, k0 + j, D)
                            : chunk_row<KT>(p, u, p.k, p.k_stride, k0 + j, D);
                if (!row) atomicMin(&s_bad, k0 + j);
                if (sizeof(KT) == 1 && row) {
                    const int id = __ldg(p.block_table + (size_t)u.b * p.max_blocks + (k0 + j) / p.page);
                    sc = __ldg((which ? p.v_scale : p.k_scale) + (long long)id * p.Hkv + u.kvh);
                }
            }
            s_rows[which][j] = row;
            s_scale[which][j] = sc;
        }
        __syncthreads();
        const bool masked = k0 + SM_KEYS > seen_by_all;
        for (int i = tid; i < 2 * SM_KEYS * D4; i += SM_THREADS) {
            const int which = i / (SM_KEYS * D4), j = i / D4 % SM_KEYS, c = i % D4;
            const KT* row = s_rows[which][j];
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (row) x = load_row4(row + 4 * c, s_scale[which][j]);
            if (which && masked && !(finite(x.x) && finite(x.y) && finite(x.z) && finite(x.w))) {
                // a row that does not see this key has probability 0 for it, and 0 x inf would be NaN:
                // such values are left out here and added at the end to the rows that see them
                s_odd = 1;
                x.x = finite(x.x) ? x.x : 0.f, x.y = finite(x.y) ? x.y : 0.f;
                x.z = finite(x.z) ? x.z : 0.f, x.w = finite(x.w) ? x.w : 0.f;
            }
            *reinterpret_cast<float4*>((which ? sv : sk) + j * C::LD + 4 * c) = x;
        }
        __syncthreads();
        float s[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll 4
        for (int c = 0; c < D4; ++c) {
            float4 a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4*>(sq + (rg + 16 * i) * C::LD + 4 * c);
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const float4*>(sk + (cg + 8 * j) * C::LD + 4 * c);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[i][j] = fmaf(a[i].x, b[j].x, s[i][j]);
                    s[i][j] = fmaf(a[i].y, b[j].y, s[i][j]);
                    s[i][j] = fmaf(a[i].z, b[j].z, s[i][j]);
                    s[i][j] = fmaf(a[i].w, b[j].w, s[i][j]);
                }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float mt = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[i][j] *= p.q_scale;
                if (k0 + cg + 8 * j >= limit[i]) s[i][j] = -INFINITY;
                mt = fmaxf(mt, s[i][j]);
            }
            const float mo = m[i];
#pragma unroll
            for (int off = 1; off < 8; off <<= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, off));
            m[i] = fmaxf(m[i], mt);
            const float mn = m[i] == -INFINITY ? 0.f : m[i];  // no key seen yet: every weight is 0
            const float w = exp2f(mo - mn);
            l[i] *= w;
#pragma unroll
            for (int c = 0; c < OC; ++c) o[i][c].x *= w, o[i][c].y *= w, o[i][c].z *= w, o[i][c].w *= w;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float e = exp2f(s[i][j] - mn);
                l[i] += e;
                sp[(rg + 16 * i) * C::LP + cg + 8 * j] = e;
            }
        }
        __syncwarp();  // a row's probabilities come from the eight lanes of its row group
#pragma unroll 2
        for (int j0 = 0; j0 < SM_KEYS; j0 += 4) {
            float4 pr[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) pr[i] = *reinterpret_cast<const float4*>(sp + (rg + 16 * i) * C::LP + j0);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int c = 0; c < OC; ++c) {
                    const float4 x = *reinterpret_cast<const float4*>(sv + (j0 + j) * C::LD + 4 * (cg + 8 * c));
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float e = j == 0 ? pr[i].x : j == 1 ? pr[i].y : j == 2 ? pr[i].z : pr[i].w;
                        o[i][c].x = fmaf(e, x.x, o[i][c].x);
                        o[i][c].y = fmaf(e, x.y, o[i][c].y);
                        o[i][c].z = fmaf(e, x.z, o[i][c].z);
                        o[i][c].w = fmaf(e, x.w, o[i][c].w);
                    }
                }
        }
    }
    __syncthreads();
    const int bad_from = s_bad;
    const bool odd = s_odd;
    if (bad_from < u.keys && tid == 0) raise_error(p.error_flag, KVB_DEVERR_BLOCK);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int off = 1; off < 8; off <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], off);
        const int r = rg + 16 * i;
        if (r >= rows) continue;
        const bool bad = bad_from < limit[i];  // the rows that see it are NaN
        if (odd && !bad) {
            const int first = max(tiles.x * SM_KEYS, seen_by_all / SM_KEYS * SM_KEYS);
            for (int j = first; j < min(limit[i], tiles.y * SM_KEYS); ++j) {
                const KT* row = chunk_row<KT>(p, u, p.v, p.v_stride, j, D);
                float sc = 1.f;
                if (sizeof(KT) == 1)
                    sc = __ldg(p.v_scale + (long long)__ldg(p.block_table + (size_t)u.b * p.max_blocks + j / p.page) *
                                               p.Hkv + u.kvh);
#pragma unroll
                for (int c = 0; c < OC; ++c) {
                    const float4 x = load_row4(row + 4 * (cg + 8 * c), sc);
                    if (!finite(x.x)) o[i][c].x += x.x;
                    if (!finite(x.y)) o[i][c].y += x.y;
                    if (!finite(x.z)) o[i][c].z += x.z;
                    if (!finite(x.w)) o[i][c].w += x.w;
                }
            }
        }
        const size_t row = (size_t)(u.row0 + r / p.G) * p.H + h0 + r % p.G;
        // (a split may hold no key that the row sees; a row whose every score is -inf is 0 / 0 = NaN)
        const float inv = bad ? __int_as_float(0x7fc00000) : p.splits > 1 && l[i] == 0.f ? 0.f : 1.f / l[i];
        if (p.splits > 1) {
            const size_t at = (size_t)u.split * p.T * p.H + row;
            if (cg == 0) p.part_ml[at] = make_float2(m[i], bad ? inv : l[i]);
#pragma unroll
            for (int c = 0; c < OC; ++c)
                *reinterpret_cast<float4*>(p.part_o + at * D + 4 * (cg + 8 * c)) =
                    make_float4(o[i][c].x * inv, o[i][c].y * inv, o[i][c].z * inv, o[i][c].w * inv);
        } else {
#pragma unroll
            for (int c = 0; c < OC; ++c) {
                QT* out = static_cast<QT*>(p.out) + row * D + 4 * (cg + 8 * c);
                if constexpr (sizeof(QT) == 4) {
                    *reinterpret_cast<float4*>(out) =
                        make_float4(o[i][c].x * inv, o[i][c].y * inv, o[i][c].z * inv, o[i][c].w * inv);
                } else {
                    *reinterpret_cast<uint2*>(out) =
                        make_uint2(h2_as_u32(__floats2half2_rn(o[i][c].x * inv, o[i][c].y * inv)),
                                   h2_as_u32(__floats2half2_rn(o[i][c].z * inv, o[i][c].w * inv)));
                }
            }
        }
    }
}

// out = sum_s l_s 2^(m_s - M) o_s / sum_s l_s 2^(m_s - M) over the splits of a row (one warp a row; D/32
// values a lane). Rows outside [cu[0], cu[B]) are not touched.
template <typename QT, int D>
__global__ void __launch_bounds__(256) chunk_merge_kernel(const __grid_constant__ ChunkParams p) {
    constexpr int E = D / 32;
    using V = typename std::conditional<E == 4, float4, float2>::type;
    const int lane = threadIdx.x & 31;
    pdl_wait();
    pdl_trigger();
    const long long rows = (long long)p.T * p.H;
    const long long first = (long long)max(0, __ldg(p.cu)) * p.H, end = min(rows, (long long)__ldg(p.cu + p.B) * p.H);
    const long long step = (long long)gridDim.x * 8;
    for (long long r = first + (long long)blockIdx.x * 8 + (threadIdx.x >> 5); r < end; r += step) {
        float M = -INFINITY, S = 0.f, A[E];
#pragma unroll
        for (int e = 0; e < E; ++e) A[e] = 0.f;
        constexpr int U = 4;
        for (int s0 = 0; s0 < p.splits; s0 += U) {
            float2 ml[U];
            V x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                ml[u] = make_float2(-INFINITY, 0.f);
                if (s0 + u < p.splits) {
                    const long long at = (long long)(s0 + u) * rows + r;
                    ml[u] = __ldcg(p.part_ml + at);
                    x[u] = __ldcg(reinterpret_cast<const V*>(p.part_o + at * D) + lane);
                }
            }
            float Mb = M;
#pragma unroll
            for (int u = 0; u < U; ++u) Mb = fmaxf(Mb, ml[u].x);
            const float c = M == Mb ? 1.f : exp2f(M - Mb);
            S *= c;
#pragma unroll
            for (int e = 0; e < E; ++e) A[e] *= c;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (ml[u].y == 0.f) continue;  // a split without keys that this row sees
                const float w = ml[u].y * exp2f(ml[u].x - Mb);
                S += w;
                const float* f = reinterpret_cast<const float*>(&x[u]);
#pragma unroll
                for (int e = 0; e < E; ++e) A[e] = fmaf(w, f[e], A[e]);
            }
            M = Mb;
        }
        const float inv = 1.f / S;
        QT* out = static_cast<QT*>(p.out) + r * D + lane * E;
        if constexpr (sizeof(QT) == 4) {
            V y;
            float* f = reinterpret_cast<float*>(&y);
#pragma unroll
            for (int e = 0; e < E; ++e) f[e] = A[e] * inv;
            *reinterpret_cast<V*>(out) = y;
        } else {
#pragma unroll
            for (int e = 0; e < E; e += 2)
                *reinterpret_cast<__half2*>(out + e) = __floats2half2_rn(A[e] * inv, A[e + 1] * inv);
        }
    }
}

// Joins the pieces of the units that the tcgen05 kernel's CTAs cut: CTA (c, y) takes the unit that part c
// began, rows 32 y .. 32 y + 31 of its two query tiles, a warp a row: the piece of part c and those of the
// parts behind it up to the unit's last.
template <typename QT, int D>
__global__ void __launch_bounds__(256) chunk_join_kernel(const __grid_constant__ ChunkParams p) {
    constexpr int E = D / 32;
    using V = typename std::conditional<E == 4, float4, float2>::type;
    const int lane = threadIdx.x & 31, c = blockIdx.x;
    pdl_wait();
    pdl_trigger();
    const ChunkPiece u = p.pieces[c];
    if (u.last < 0) return;
#pragma unroll 1
    for (int i = threadIdx.x >> 5; i < 32; i += 8) {
        const int rr = blockIdx.y * 32 + i, t = rr / 128, r = rr % 128;
        const int tok = t * p.tile_tokens + r / p.G;
        if (r >= p.tile_tokens * p.G || tok >= u.n) continue;
        float M = -INFINITY, S = 0.f, A[E];
#pragma unroll
        for (int e = 0; e < E; ++e) A[e] = 0.f;
        constexpr int U = 4;
        for (int k0 = c; k0 <= u.last; k0 += U) {
            float2 ml[U];
            V x[U];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int k = k0 + j;
                ml[j] = make_float2(-INFINITY, 0.f);
                if (k <= u.last && (k == c || p.pieces[k].head)) {
                    const long long at = ((long long)(k == c ? 2 * k + 1 : 2 * k) * 2 + t) * 128 + r;
                    ml[j] = __ldcg(p.part_ml + at);
                    x[j] = __ldcg(reinterpret_cast<const V*>(p.part_o + at * D) + lane);
                }
            }
            float Mb = M;
#pragma unroll
            for (int j = 0; j < U; ++j) Mb = fmaxf(Mb, ml[j].x);
            const float sc = M == Mb ? 1.f : exp2f(M - Mb);
            S *= sc;
#pragma unroll
            for (int e = 0; e < E; ++e) A[e] *= sc;
#pragma unroll
            for (int j = 0; j < U; ++j) {
                if (ml[j].y == 0.f) continue;  // a piece without keys that this row sees
                const float w = ml[j].y * exp2f(ml[j].x - Mb);
                S += w;
                const float* f = reinterpret_cast<const float*>(&x[j]);
#pragma unroll
                for (int e = 0; e < E; ++e) A[e] = fmaf(w, f[e], A[e]);
            }
            M = Mb;
        }
        const float inv = 1.f / S;
        QT* out = static_cast<QT*>(p.out) + ((size_t)(u.row0 + tok) * p.H + u.kvh * p.G + r % p.G) * D + lane * E;
        if constexpr (sizeof(QT) == 4) {
            V y;
            float* f = reinterpret_cast<float*>(&y);
#pragma unroll
            for (int e = 0; e < E; ++e) f[e] = A[e] * inv;
            *reinterpret_cast<V*>(out) = y;
        } else {
#pragma unroll
            for (int e = 0; e < E; e += 2)
                *reinterpret_cast<__half2*>(out + e) = __floats2half2_rn(A[e] * inv, A[e + 1] * inv);
        }
    }
}

template <typename QT, typename KT, int D>
cudaError_t launch(const ChunkParams& p, cudaStream_t stream) {
    using C = SimtCfg<D>;
    static KvbPerDevice<int> configured;
    int done = 0;
    cudaError_t e = configured.get(&done, [](int* v) {
        *v = 1;
        return cudaFuncSetAttribute(chunk_simt_kernel<QT, KT, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    int(C::SMEM));
    });
    if (e != cudaSuccess) return e;
    return kvb_launch_pdl(chunk_simt_kernel<QT, KT, D>, (unsigned)p.units, SM_THREADS, C::SMEM, stream, p);
}

template <typename QT, typename KT>
cudaError_t launch_d(const ChunkParams& p, int D, cudaStream_t stream) {
    return D == 128 ? launch<QT, KT, 128>(p, stream) : launch<QT, KT, 64>(p, stream);
}

}  // namespace

cudaError_t kvb_launch_chunk_simt(const ChunkParams& p, int q_type, int kv_type, int D, cudaStream_t stream) {
    if (q_type == KVB_F32)
        return kv_type == KVB_F32   ? launch_d<float, float>(p, D, stream)
               : kv_type == KVB_F16 ? launch_d<float, __half>(p, D, stream)
                                    : launch_d<float, int8_t>(p, D, stream);
    return kv_type == KVB_F32   ? launch_d<__half, float>(p, D, stream)
           : kv_type == KVB_F16 ? launch_d<__half, __half>(p, D, stream)
                                : launch_d<__half, int8_t>(p, D, stream);
}

cudaError_t kvb_launch_chunk_merge(const ChunkParams& p, int q_type, int D, int num_sms, cudaStream_t stream) {
    const long long rows = (long long)p.T * p.H;
    const unsigned grid = (unsigned)std::max<long long>(1, std::min<long long>((rows + 7) / 8, (long long)num_sms * 8));
    if (q_type == KVB_F32)
        return D == 128 ? kvb_launch_pdl(chunk_merge_kernel<float, 128>, grid, 256, 0, stream, p)
                        : kvb_launch_pdl(chunk_merge_kernel<float, 64>, grid, 256, 0, stream, p);
    return D == 128 ? kvb_launch_pdl(chunk_merge_kernel<__half, 128>, grid, 256, 0, stream, p)
                    : kvb_launch_pdl(chunk_merge_kernel<__half, 64>, grid, 256, 0, stream, p);
}

cudaError_t kvb_launch_chunk_join(const ChunkParams& p, int q_type, int D, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    // 32 rows a CTA; where no sequence fills a query tile, only the rows that can hold a token
    const int rows = p.max_new <= p.tile_tokens ? p.max_new * p.G : 256;
    cfg.gridDim = dim3((unsigned)p.ctas, (unsigned)((rows + 31) / 32));
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (q_type == KVB_F32)
        return D == 128 ? cudaLaunchKernelEx(&cfg, chunk_join_kernel<float, 128>, p)
                        : cudaLaunchKernelEx(&cfg, chunk_join_kernel<float, 64>, p);
    return D == 128 ? cudaLaunchKernelEx(&cfg, chunk_join_kernel<__half, 128>, p)
                    : cudaLaunchKernelEx(&cfg, chunk_join_kernel<__half, 64>, p);
}
