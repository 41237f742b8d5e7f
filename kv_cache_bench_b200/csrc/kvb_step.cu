// The two steps in front of attention when a serving step adds several tokens per sequence:
//
//   plan    which physical page and slot every new token of the step gets. With len_b tokens cached
//           and n_b new ones, pages of P tokens:
//             cu_b   = n_0 + ... + n_(b-1)                    (where b's tokens start in the packed step)
//             have_b = ceil(len_b / P), need_b = ceil((len_b + n_b) / P) - have_b
//             E_b    = need_0 + ... + need_b
//           Sequence b's i-th new page is free id ring[(head + E_b - need_b + i) mod ring_size]; a
//           sequence is served when its pages fit (need_b = 0 or E_b <= tail - head), so the served
//           sequences that need pages are the first ones, and the result does not depend on timing.
//   append  the new tokens' K and V rows written into those pages (fp32, fp16), or quantized into
//           int8 pages with one scale per (page, KV head).
//
// No counterpart in the reference, whose block tables are built on the host before the run
// (src/reference.cpp:11-30) and whose caches are written whole (src/reference.hpp:60-68,
// src/reference.cpp:32-51).
#include <cuda_fp16.h>

#include <algorithm>

#include "kvb_quant.cuh"
#include "kvb_step.h"

namespace {

using namespace kvb_dev;

// ---- plan ---------------------------------------------------------------------------------------

constexpr int PL_THREADS = 512;
constexpr int PL_WARPS = PL_THREADS / 32;

struct Pair {
    long long tok, blk;
};

// Every CTA scans the lengths (one sequence per thread and round) and then writes the slots of its own
// range of tokens; CTA 0 also writes what belongs to the sequences. Nothing passes between CTAs, so
// one launch does it all and B lengths are read once per CTA from L2. Bound by latency: two dependent
// loads, a block scan and a store.
__global__ void __launch_bounds__(PL_THREADS) step_plan_kernel(const PlanParams p) {
    __shared__ int s_cu[PL_THREADS + 1];        // first token of a sequence of this round
    __shared__ int s_len[PL_THREADS], s_have[PL_THREADS];
    __shared__ long long s_first[PL_THREADS];   // ring position of its first new page; -1: not served
    __shared__ Pair s_warp[PL_WARPS];
    __shared__ unsigned long long s_head;
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    pdl_wait();
    pdl_trigger();
    long long head = __ldg(p.ring_pos), avail = __ldg(p.ring_pos + 1) - head;
    if (head < 0 || avail < 0 || avail > p.ring_size) {
        if (blockIdx.x == 0 && tid == 0 && p.error_flag) raise_error(p.error_flag, KVB_DEVERR_STATE);
        head = max(head, 0ll);
        avail = 0;
    }
    const long long head0 = p.ring_size > 0 ? head % p.ring_size : 0;
    const long long capacity = min((long long)p.max_blocks * p.page, 0x7fffffffll);
    const int per = int(((long long)p.num_tokens + gridDim.x - 1) / gridDim.x);
    const int t0 = int(min((long long)p.num_tokens, (long long)blockIdx.x * per));
    const int t1 = int(min((long long)p.num_tokens, (long long)t0 + per));
    if (tid == 0) s_head = 0;
    long long tok = 0, blk = 0;  // totals of the rounds before
    unsigned bad = 0;
    for (int b0 = 0; b0 < p.B; b0 += PL_THREADS) {
        if (blockIdx.x != 0 && tok >= t1) break;
        const int b = b0 + tid;
        int len = 0, n = 0, have = 0, need = 0;
        bool valid = false;
        if (b < p.B) {
            len = __ldg(p.seq_lens + b);
            n = __ldg(p.new_lens + b);
            valid = len >= 0 && n >= 0 && (long long)len + n <= capacity;
            n = max(n, 0);
            if (valid) {
                have = len == 0 ? 0 : kvb_div(len - 1, p.div_page) + 1;
                need = (len + n == 0 ? 0 : kvb_div(len + n - 1, p.div_page) + 1) - have;
            }
        }
        Pair v{n, need};
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long a = __shfl_up_sync(0xffffffffu, v.tok, o), c = __shfl_up_sync(0xffffffffu, v.blk, o);
            if (lane >= o) v.tok += a, v.blk += c;
        }
        __syncthreads();  // the round before is done with the shared arrays
        if (lane == 31) s_warp[w] = v;
        __syncthreads();
        long long all_tok = 0, all_blk = 0;
#pragma unroll
        for (int i = 0; i < PL_WARPS; ++i) {
            const Pair x = s_warp[i];
            if (i < w) v.tok += x.tok, v.blk += x.blk;
            all_tok += x.tok, all_blk += x.blk;
        }
        const long long end = tok + v.tok, start = end - n;  // exclusive and inclusive token sums
        const long long E = blk + v.blk;
        const bool served = valid && end <= p.num_tokens && (need == 0 || E <= avail);
        const int cut = int(min(start, (long long)p.num_tokens));
        s_cu[tid] = cut;
        s_len[tid] = valid ? len : 0;
        s_have[tid] = have;
        s_first[tid] = served ? E - need : -1;
        if (tid == PL_THREADS - 1) s_cu[PL_THREADS] = int(min(end, (long long)p.num_tokens));
        if (blockIdx.x == 0 && b < p.B) {
            p.total_lens[b] = served ? len + n : -1;
            p.cu_new[b] = cut;
            if (b == p.B - 1) p.cu_new[p.B] = int(min(end, (long long)p.num_tokens));
            if (!valid || end > p.num_tokens) bad |= KVB_DEVERR_LENGTH;
            else if (!served) bad |= KVB_DEVERR_BLOCK;
            if (served && need > 0) atomicMax(&s_head, (unsigned long long)E);
        }
        __syncthreads();
        // this round's tokens in the CTA's range
        const int a = max(t0, int(min(tok, (long long)p.num_tokens)));
        const int z = min(t1, int(min(tok + all_tok, (long long)p.num_tokens)));
        for (int t = a + tid; t < z; t += PL_THREADS) {
            int lo = 0, hi = PL_THREADS - 1;  // the last sequence that starts at or before t
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (s_cu[mid] <= t) lo = mid;
                else hi = mid - 1;
            }
            const int pos = s_len[lo] + (t - s_cu[lo]);
            const long long first = s_first[lo];
            long long slot = -1;
            if (first >= 0) {
                const int pg = kvb_div(pos, p.div_page), at = pos - pg * p.page, fresh = pg - s_have[lo];
                int* entry = p.block_table + (size_t)(b0 + lo) * p.max_blocks + pg;
                int id;
                if (fresh >= 0) {
                    long long r = head0 + first + fresh;  // below twice the ring's size
                    if (r >= p.ring_size) r -= p.ring_size;
                    id = __ldg(p.ring + r);
                    if (at == 0) *entry = id;
                } else {
                    id = *entry;
                }
                if (id >= 0 && id < p.num_blocks) slot = (long long)id * p.page + at;
                else bad |= KVB_DEVERR_BLOCK;
            }
            p.slot_map[t] = slot;
            if (p.positions) p.positions[t] = pos;
        }
        tok += all_tok;
        blk += all_blk;
    }
    // entries behind the last token
    for (long long t = max((long long)t0, tok) + tid; t < t1; t += PL_THREADS) {
        p.slot_map[t] = -1;
        if (p.positions) p.positions[t] = 0;
    }
    if (blockIdx.x == 0) {
        __syncthreads();
        if (tid == 0) {
            p.ring_out[0] = __ldg(p.ring_pos) + (long long)s_head;
            p.ring_out[1] = __ldg(p.ring_pos + 1);
            if (p.B == 0) p.cu_new[0] = 0;
        }
    }
    if (bad && p.error_flag) raise_error(p.error_flag, bad);
}

// ---- append -------------------------------------------------------------------------------------

constexpr int AP_THREADS = 256;
constexpr int AP_UNROLL = 4;  // pieces in flight per thread

// fp32 and fp16 pools: a warp moves one token's K (or V) rows, in pieces of 16 destination bytes, several per
// lane in flight; a token's rows are contiguous in the source and each head's row in the pool. The slot is
// read and divided once per token. Bound by memory. (One piece per thread over the whole step, with its place
// found by divisions: 72-80 us for 21 k fp32 tokens of 8 x 128 into fp16 pages.)
template <typename SRC, typename DST>
__global__ void __launch_bounds__(AP_THREADS) append_rows_kernel(const AppendParams p) {
    constexpr int PER = 16 / sizeof(DST);  // values per piece
    constexpr int N = sizeof(SRC) / sizeof(DST) > 1 ? 2 : 1;
    const int which = blockIdx.y, lane = threadIdx.x & 31;
    const SRC* src = static_cast<const SRC*>(p.src[which]);
    DST* pool = static_cast<DST*>(p.pool[which]);
    const int pieces = p.Hkv * int(p.div_row.d);  // of a token, below 2^31 (checked by the host)
    const long long limit = p.num_blocks * p.page;
    pdl_wait();
    pdl_trigger();
    const int step = gridDim.x * (AP_THREADS / 32);
    for (long long t = blockIdx.x * (AP_THREADS / 32) + (threadIdx.x >> 5); t < p.num_tokens; t += step) {
        const long long slot = __ldg(p.slot_map + t);
        if (slot < 0 || slot >= limit) {
            if (slot != -1 && p.error_flag && lane == 0) raise_error(p.error_flag, KVB_DEVERR_BLOCK);
            continue;
        }
        const long long block = slot < (1ll << 31) ? kvb_div(int(slot), p.div_page) : slot / p.page;
        const int at = int(slot - block * p.page);
        const SRC* row = src + t * p.stride[which];
        DST* to = pool + (block * p.Hkv * p.page + at) * p.D;  // head 0's row; the others page rows apart
        for (int c0 = lane; c0 < pieces; c0 += 32 * AP_UNROLL) {
            uint4 raw[AP_UNROLL][N];
#pragma unroll
            for (int u = 0; u < AP_UNROLL; ++u) {
                const int c = c0 + 32 * u;
                if (c >= pieces) continue;
                const uint4* s = reinterpret_cast<const uint4*>(row + (long long)c * PER);
                raw[u][0] = __ldcs(s);
                if constexpr (N > 1) raw[u][1] = __ldcs(s + 1);
            }
#pragma unroll
            for (int u = 0; u < AP_UNROLL; ++u) {
                const int c = c0 + 32 * u;
                if (c >= pieces) continue;
                const int h = kvb_div(c, p.div_row), in = c - h * int(p.div_row.d);
                uint4 out = raw[u][0];
                if constexpr (N > 1) {  // fp32 rows into fp16 pages: one rounding to nearest
                    const float4 f = *reinterpret_cast<const float4*>(&raw[u][0]);
                    const float4 g = *reinterpret_cast<const float4*>(&raw[u][N - 1]);
                    out = make_uint4(h2_as_u32(__floats2half2_rn(f.x, f.y)), h2_as_u32(__floats2half2_rn(f.z, f.w)),
                                     h2_as_u32(__floats2half2_rn(g.x, g.y)), h2_as_u32(__floats2half2_rn(g.z, g.w)));
                }
                *reinterpret_cast<uint4*>(to + (long long)h * p.page * p.D + in * PER) = out;
            }
        }
    }
}

template <typename SRC>
__device__ __forceinline__ float4 load4(const SRC* s) {
    if constexpr (sizeof(SRC) == 4) {
        return __ldg(reinterpret_cast<const float4*>(s));
    } else {
        const uint2 r = __ldg(reinterpret_cast<const uint2*>(s));
        const float2 a = __half22float2(u32_as_h2(r.x)), b = __half22float2(u32_as_h2(r.y));
        return make_float4(a.x, a.y, b.x, b.y);
    }
}

// Larger of the two, NaN if one is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

__device__ __forceinline__ float amax4(float4 v) {
    return max_nan(max_nan(fabsf(v.x), fabsf(v.y)), max_nan(fabsf(v.z), fabsf(v.w)));
}

// int8 pools. A run is the new tokens of one sequence that share a page, for one KV head of K or V, and TPR
// threads (a warp, or the CTA for pages of 32 KB of fp32 and more) take it. The page's scale becomes
// s = max(s_old, amax / 127) (s_old only if the page had rows before); rows that were there are rounded
// again, rint(q * (s_old / s)), when the scale grew; new rows by the page quantizer's rule (kvb_quant.cuh). A
// NaN among the rows makes amax and s NaN (rows 0), and a scale that is not finite stays until the page is begun
// anew, so that no value which is not finite turns into a number. A token starts a run if it is its sequence's first new one or the first of its page; each group looks for
// them among `tpg` tokens. A run of up to AP_REGS float4 per thread stays in registers between the maximum
// and the rounding, a larger one is read again (from L1 or L2). Bound by memory; with a warp for every run
// and two reads, prompts of 7 k tokens into pages of 128 took 120 us.
constexpr int AP_REGS = 16;

template <typename SRC, int TPR>
__global__ void __launch_bounds__(AP_THREADS, 3) append_i8_kernel(const AppendParams p, int tpg,
                                                                int heads) {
    constexpr int WARPS = TPR / 32;
    __shared__ int s_tok[AP_THREADS], s_n[AP_THREADS], s_at[AP_THREADS];  // a CTA-wide group's runs
    __shared__ long long s_block[AP_THREADS];
    __shared__ int s_runs;
    __shared__ float s_max[2][AP_THREADS / 32];
    const int lane = threadIdx.x & 31, gl = threadIdx.x % TPR;
    // The heads of a token group are neighbours in the grid, so that CTAs that run together read whole rows.
    const int by = int(blockIdx.x % heads);
    const long long tok0 = ((long long)(blockIdx.x / heads) * (AP_THREADS / TPR) + threadIdx.x / TPR) * tpg;
    pdl_wait();
    pdl_trigger();
    // each of the first tpg threads of a group decodes one token
    const int t = int(min(tok0 + gl, (long long)p.num_tokens));
    int n = 0, at = 0;
    long long block = -1;
    if (gl < tpg && t < p.num_tokens) {
        int lo = 0, hi = p.B;  // the first sequence that ends behind t
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (__ldg(p.cu_new + mid + 1) > t) hi = mid;
            else lo = mid + 1;
        }
        if (lo < p.B) {
            const int c0 = __ldg(p.cu_new + lo), c1 = min(__ldg(p.cu_new + lo + 1), p.num_tokens);
            const int total = __ldg(p.total_lens + lo);
            const long long start = (long long)total - (__ldg(p.cu_new + lo + 1) - c0);
            if (c0 >= 0 && c0 <= t) {
                if (start < 0 || (long long)total > (long long)p.max_blocks * p.page) {
                    // -1 marks a sequence that the plan refused: it was reported there
                    if (total != -1 && t == c0 && by == 0 && p.error_flag)
                        raise_error(p.error_flag, KVB_DEVERR_LENGTH);
                } else {
                    const int pos = int(start) + (t - c0), pg = kvb_div(pos, p.div_page);
                    at = pos - pg * p.page;
                    if (t == c0 || at == 0) {
                        const int id = __ldg(p.block_table + (size_t)lo * p.max_blocks + pg);
                        if (id >= 0 && id < p.num_blocks) {
                            block = id;
                            n = min(p.page - at, c1 - t);
                        } else if (by == 0 && p.error_flag) {
                            raise_error(p.error_flag, KVB_DEVERR_BLOCK);
                        }
                    }
                }
            }
        }
    }
    const int dw = int(p.div_row.d);  // pieces of four values per row
    int parity = 0;  // alternates the CTA-wide reduction's slots
    auto run = [&](int y, int rt, int rn, int rat, long long rblock) {
        const int h = y >> 1, which = y & 1;
        const SRC* src = static_cast<const SRC*>(p.src[which]) + (long long)h * p.D;
        const long long stride = p.stride[which];
        const long long rb = rblock * p.Hkv + h;
        const SRC* rows = src + rt * stride;
        uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<int8_t*>(p.pool[which]) + rb * p.page * p.D);
        const int pieces = rn * dw;  // below 2^31: a page of one head is (checked by the host)
        const bool keep = pieces <= TPR * AP_REGS;
        float4 v[AP_REGS];
        float amax = 0.f;
        auto load = [&](int i0) {
#pragma unroll
            for (int u = 0; u < AP_REGS; ++u) {
                const int i = i0 + TPR * u;
                v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i < pieces) {
                    const int r = kvb_div(i, p.div_row);
                    v[u] = load4(rows + r * stride + 4 * (i - r * dw));
                }
            }
        };
        for (int i0 = gl; i0 < pieces; i0 += TPR * AP_REGS) {
            load(i0);
#pragma unroll
            for (int u = 0; u < AP_REGS; ++u) amax = max_nan(amax, amax4(v[u]));
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if constexpr (WARPS > 1) {
            if (lane == 0) s_max[parity][threadIdx.x >> 5] = amax;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < WARPS; ++i) amax = max_nan(amax, s_max[parity][i]);
            parity ^= 1;
        }
        float scale = amax / 127.0f;
        if (rat > 0) {
            const float old = p.scale[which][rb];
            if (scale == scale && !(old < scale)) {  // (old may be NaN)
                scale = old;
            } else {
                const float ratio = __fdiv_rn(old, scale);
                for (int i = gl; i < rat * dw; i += TPR) {
                    const uint32_t x = dst[i];
                    uint32_t y = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int q = __float2int_rn(__fmul_rn(float(int8_t(x >> (8 * e))), ratio));
                        y |= uint32_t(q & 255) << (8 * e);
                    }
                    dst[i] = y;
                }
            }
        }
        if constexpr (WARPS > 1) __syncthreads();  // every thread has read the old scale
        else __syncwarp();
        if (gl == 0) p.scale[which][rb] = scale;
        dst += rat * dw;
        const float rcp = finite_rcp(scale);
        for (int i0 = gl; i0 < pieces; i0 += TPR * AP_REGS) {
            if (!keep) load(i0);
            int near = scale > 0.f && rcp == 0.f;
#pragma unroll
            for (int u = 0; u < AP_REGS; ++u) {
                const int i = i0 + TPR * u;
                if (i < pieces) dst[i] = scale > 0.f ? quantize4_fast(v[u], rcp, near) : 0u;
            }
            if (near) {
#pragma unroll
                for (int u = 0; u < AP_REGS; ++u) {
                    const int i = i0 + TPR * u;
                    if (i < pieces) dst[i] = quantize4_exact(v[u], scale);
                }
            }
        }
    };
    if constexpr (WARPS > 1) {
        if (threadIdx.x == 0) s_runs = 0;
        __syncthreads();
        if (block >= 0) {
            const int i = atomicAdd(&s_runs, 1);  // (their order does not matter: a page has one run)
            s_tok[i] = t, s_n[i] = n, s_at[i] = at, s_block[i] = block;
        }
        __syncthreads();
        for (int y = by; y < 2 * p.Hkv; y += heads)
            for (int i = 0; i < s_runs; ++i) run(y, s_tok[i], s_n[i], s_at[i], s_block[i]);
    } else {
        for (unsigned runs = __ballot_sync(0xffffffffu, block >= 0); runs; runs &= runs - 1) {
            const int l = __ffs(runs) - 1;
            const int rt = __shfl_sync(0xffffffffu, t, l), rn = __shfl_sync(0xffffffffu, n, l);
            const int rat = __shfl_sync(0xffffffffu, at, l);
            const long long rblock = __shfl_sync(0xffffffffu, block, l);
            for (int y = by; y < 2 * p.Hkv; y += heads) run(y, rt, rn, rat, rblock);
        }
    }
}

template <typename SRC, typename DST>
cudaError_t launch_rows(const AppendParams& p, int num_sms, cudaStream_t stream) {
    const long long ctas = std::min<long long>(((long long)p.num_tokens + AP_THREADS / 32 - 1) / (AP_THREADS / 32),
                                               (long long)num_sms * 8);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)std::max<long long>(1, ctas), 2);
    cfg.blockDim = dim3(AP_THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, append_rows_kernel<SRC, DST>, p);
}

template <typename SRC>
cudaError_t launch_i8(const AppendParams& p, int num_sms, cudaStream_t stream) {
    // A CTA for every run where a page of one head is large and the step mean is more than a few rows a
    // sequence; it looks at 128 tokens. Otherwise a warp, which looks at one token while that keeps the grid
    // small, up to 32 (most are no run's first).
    const bool cta = (long long)p.page * p.D * 4 >= 32768 && p.num_tokens >= 8ll * p.B;
    int tpg = cta ? 128 : 1;
    if (!cta)
        while (tpg < 32 && (long long)p.num_tokens / tpg * p.Hkv * 2 > (long long)num_sms * 64) tpg *= 2;
    const long long groups = ((long long)p.num_tokens + tpg - 1) / tpg, per = cta ? 1 : AP_THREADS / 32;
    cudaLaunchConfig_t cfg = {};
    // heads of K and V side by side, as many as make six CTAs an SM; a CTA does the others after them, with the
    // runs that it found once
    const long long x = (groups + per - 1) / per;
    const long long y = std::min<long long>(2ll * p.Hkv, std::max<long long>(1, (6ll * num_sms + x - 1) / x));
    if (x * y >= (1ll << 31)) return cudaErrorInvalidConfiguration;
    cfg.gridDim = dim3((unsigned)(x * y));
    cfg.blockDim = dim3(AP_THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cta ? cudaLaunchKernelEx(&cfg, append_i8_kernel<SRC, AP_THREADS>, p, tpg, int(y))
               : cudaLaunchKernelEx(&cfg, append_i8_kernel<SRC, 32>, p, tpg, int(y));
}

}  // namespace

cudaError_t kvb_launch_step_plan(const PlanParams& p, int num_sms, cudaStream_t stream) {
    // 1024 tokens per CTA (two per thread): enough CTAs to spread a prompt's slots, one for a decode step
    const long long ctas = std::min<long long>(((long long)p.num_tokens + 1023) / 1024, 2ll * num_sms);
    return kvb_launch_pdl(step_plan_kernel, (unsigned)std::max<long long>(1, ctas), PL_THREADS, 0, stream, p);
}

cudaError_t kvb_launch_append(const AppendParams& p, int src_type, int kv_type, int num_sms, cudaStream_t stream) {
    if (kv_type == KVB_I8)
        return src_type == KVB_F32 ? launch_i8<float>(p, num_sms, stream) : launch_i8<__half>(p, num_sms, stream);
    if (kv_type == KVB_F32) return launch_rows<float, float>(p, num_sms, stream);
    return src_type == KVB_F32 ? launch_rows<float, __half>(p, num_sms, stream)
                               : launch_rows<__half, __half>(p, num_sms, stream);
}
