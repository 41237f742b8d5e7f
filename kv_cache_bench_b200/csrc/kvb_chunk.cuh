// Attention of several new tokens per sequence: what the tcgen05 kernel (kvb_chunk_umma.cu), the
// CUDA-core kernel and the merge of split keys (kvb_chunk_simt.cu) share.
//
// A call has `B` sequences whose new tokens are packed: sequence b owns query rows cu[b] .. cu[b+1) of
// q and out ([T][H][D]). Its keys and values are total_b tokens long, in pages found through the block
// table, or (whole prompts) the packed rows cu[b] .. cu[b+1) of contiguous k and v. New token i of b
// sits at position ctx_b + i, ctx_b = total_b - n_b, and sees the tokens at positions <= its own:
//     out[i][h] = sum_j softmax_j(q[i][h] . k[j][h / G] / sqrt(D)) v[j][h / G].
#pragma once

#include "kvb_device.cuh"
#include "kvb_step.h"

struct ChunkParams {
    const void* q;              // [T][H][D], fp32 or fp16; q_stride elements between tokens
    void* out;                  // [T][H][D], q's type
    const void* k;              // pools [num_blocks][Hkv][page][D], or packed [T][Hkv][D]
    const void* v;
    long long q_stride, k_stride, v_stride;  // elements between tokens (k, v: packed only)
    const float* k_scale;       // int8 pools: [num_blocks][Hkv]
    const float* v_scale;
    const int* block_table;     // [B][max_blocks]; null: packed keys and values
    const int* total_lens;      // [B] (pages only)
    const int* cu;              // [B + 1]
    unsigned* error_flag;
    float* part_o;              // splits > 1: [splits][T][H][D], each split's normalized output
    float2* part_ml;            // [splits][T][H]: (max in log2 units, sum); a NaN sum: refused
                                // tcgen05 kernel: [2 ctas][2 tiles][128 rows] ([D]): the CTAs' partial units
    float* fold;                // tcgen05 kernel, long keys: each CTA's running sums [2 tiles][D / 4][128][4]
    struct ChunkPiece* pieces;  // tcgen05 kernel: [ctas]
    int ctas;                   // tcgen05 kernel: CTAs that share the work
    long long num_blocks;
    int B, H, Hkv, G, T;
    int page, max_blocks, max_new, max_len;
    int tile_tokens;            // new tokens of one query tile (tile rows / G)
    int unit_tokens;            // new tokens of one unit (one or two tiles)
    int blocks_of_new;          // units along the new tokens of the longest sequence
    int splits;                 // parts that a unit's keys are split into
    long long units;            // blocks_of_new * B * splits * Hkv
    float q_scale;              // log2(e) / sqrt(D)
};

// Key tiles of 128 after which the tcgen05 kernel adds its fp32 (fp16) results' sums into `fold`.
#define KVB_CHUNK_FOLD_F32 12
#define KVB_CHUNK_FOLD_F16 64

// What a CTA of the tcgen05 kernel leaves for the merge: the unit whose first keys it took and whose others
// the next CTAs did, and whether it took later keys of a unit that an earlier CTA began.
struct ChunkPiece {
    int kvh, row0, n;  // the unit: KV head, first token, tokens
    int last;          // last CTA with keys of it; -1: this CTA began no such unit
    int head;          // it has such later keys
};

// Whether the tcgen05 kernel takes the call.
bool kvb_chunk_umma_supported(int q_type, int kv_type, bool paged, int D, int page, int G);
cudaError_t kvb_launch_chunk_umma(const ChunkParams& p, int q_type, int kv_type, int D, const void* tmap_q,
                                  const void* tmap_k, const void* tmap_v, cudaStream_t stream);
cudaError_t kvb_launch_chunk_simt(const ChunkParams& p, int q_type, int kv_type, int D, cudaStream_t stream);
cudaError_t kvb_launch_chunk_merge(const ChunkParams& p, int q_type, int D, int num_sms, cudaStream_t stream);
cudaError_t kvb_launch_chunk_join(const ChunkParams& p, int q_type, int D, cudaStream_t stream);
// New tokens and units of the two kernels' query tiles.
constexpr int KVB_SIMT_ROWS = 64;

namespace kvb_dev {

// One unit of work: up to unit_tokens new tokens of one sequence, the query heads of one KV head, and
// one part of the keys they see.
struct ChunkUnit {
    int b, kvh, split;
    int row0;      // first packed query row (token)
    int n;         // new tokens of the unit
    int pos0;      // position of the first one
    int keys;      // keys of the sequence that the unit's last token sees
    int kv0;       // first packed key row (prompts)
    int state;     // 0: work, 1: no unit here, 2: refused: rows [row0, row0 + n) become NaN
};

// A sequence's place in a call, checked.
struct ChunkSeq {
    int c0, n, ctx;  // first packed row, new tokens, keys before them
    bool bad;
};

__device__ __forceinline__ ChunkSeq chunk_seq(const ChunkParams& p, int b) {
    const int c0 = __ldg(p.cu + b), c1 = __ldg(p.cu + b + 1);
    const long long n = (long long)c1 - c0;
    const long long total = p.block_table ? __ldg(p.total_lens + b) : n;
    ChunkSeq s;
    s.bad = c0 < 0 || n < 0 || c1 > p.T || n > p.max_new || (n > 0 && total < n) || total > p.max_len ||
            (p.block_table && total > (long long)p.max_blocks * p.page);
    s.c0 = c0;
    s.n = int(n);
    s.ctx = int(total - n);
    if (s.bad) {
        s.c0 = min(max(c0, 0), p.T);
        s.n = max(0, min(max(c1, 0), p.T) - s.c0);
        s.ctx = 0;
    }
    return s;
}

// Units are numbered with the last tokens of the sequences first: they see the most keys, so the
// longest units start first and the short ones fill the end.
__device__ __forceinline__ ChunkUnit chunk_unit(const ChunkParams& p, long long idx) {
    ChunkUnit u;
    u.kvh = int(idx % p.Hkv);
    long long r = idx / p.Hkv;
    u.split = int(r % p.splits);
    r /= p.splits;
    u.b = int(r % p.B);
    const int blk = p.blocks_of_new - 1 - int(r / p.B);
    const ChunkSeq s = chunk_seq(p, u.b);
    u.row0 = u.kv0 = s.c0;
    u.state = 1;
    u.n = u.pos0 = u.keys = 0;
    if (s.bad) {
        if (blk != 0) return u;
        u.state = 2;
        u.n = s.n;
        return u;
    }
    const int t0 = blk * p.unit_tokens;
    if (t0 >= s.n) return u;
    u.state = 0;
    u.row0 = s.c0 + t0;
    u.n = min(p.unit_tokens, s.n - t0);
    u.pos0 = s.ctx + t0;
    u.keys = u.pos0 + u.n;
    return u;
}

// Key tiles [first, second) of a unit that its split takes: even parts of the tiles it sees.
__device__ __forceinline__ int2 chunk_split_tiles(const ChunkParams& p, const ChunkUnit& u, int tile) {
    const int nt = (u.keys + tile - 1) / tile;
    return make_int2(int((long long)nt * u.split / p.splits), int((long long)nt * (u.split + 1) / p.splits));
}

// A refused sequence's rows become NaN (every split writes its own share), by `nthreads` threads.
template <typename QT, int D>
__device__ __forceinline__ void chunk_refuse(const ChunkParams& p, const ChunkUnit& u, int tid, int nthreads) {
    const float nanv = __int_as_float(0x7fc00000);
    const int h0 = u.kvh * p.G;
    for (long long i = tid; i < (long long)u.n * p.G; i += nthreads) {
        const size_t row = (size_t)(u.row0 + int(i / p.G)) * p.H + h0 + int(i % p.G);
        if (p.splits > 1) {
            p.part_ml[(size_t)u.split * p.T * p.H + row] = make_float2(NEG_BIG, nanv);
        } else {
            QT* o = static_cast<QT*>(p.out) + row * D;
            for (int d = 0; d < D; ++d) o[d] = QT(nanv);
        }
    }
    if (tid == 0 && u.split == 0 && u.kvh == 0) raise_error(p.error_flag, KVB_DEVERR_LENGTH);
}

// First element of key row `pos` (position in the sequence) of the unit's KV head, in the pool or the
// packed rows; null when its page's id is refused.
template <typename T>
__device__ __forceinline__ const T* chunk_row(const ChunkParams& p, const ChunkUnit& u, const void* base,
                                              long long stride, int pos, int D) {
    if (!p.block_table) return static_cast<const T*>(base) + (long long)(u.kv0 + pos) * stride + (long long)u.kvh * D;
    const int pg = pos / p.page;
    const int id = __ldg(p.block_table + (size_t)u.b * p.max_blocks + pg);
    if (id < 0 || id >= p.num_blocks) return nullptr;
    return static_cast<const T*>(base) + (((long long)id * p.Hkv + u.kvh) * p.page + (pos - pg * p.page)) * D;
}

}  // namespace kvb_dev
