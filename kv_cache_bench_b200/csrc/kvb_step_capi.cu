// Host side of the serving-step entry points of include/kvb_cuda.h: argument checks, the grid's
// geometry, tensor maps and launches. Nothing is read on the host or kept from one call for the next.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "kvb_chunk.cuh"

namespace {

int invalid(const char* msg) { return kvb_fail(KVB_ERR_INVALID, msg); }

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

bool aligned32(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31u) == 0; }

int elem_size(int t) { return t == KVB_F32 ? 4 : t == KVB_F16 ? 2 : 1; }

int launched(cudaError_t e) { return e == cudaSuccess ? KVB_OK : kvb_fail(KVB_ERR_DEVICE, cudaGetErrorString(e)); }

bool overlap(const void* a, size_t na, const void* b, size_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && na && nb && x < y + nb && y < x + na;
}

// A token's row of `heads` x D elements at `base`, `stride` elements apart, read in 16-byte pieces.
int check_rows(const void* base, int64_t stride, int64_t row, int elem, int num_tokens) {
    if (!base) return invalid("null device pointer");
    if (!aligned16(base)) return invalid("rows must be 16-byte aligned");
    if (num_tokens > 1 && (stride < row || (stride * elem) % 16 != 0))
        return invalid("a token stride must hold a whole row and be a multiple of 16 bytes");
    return KVB_OK;
}

// What both attention entry points have in common, in one form.
struct Attend {
    kvb_shape s;
    int q_type, kv_type, kernel;
    bool paged;
    ChunkParams p;
    int64_t workspace, pieces_off, ml_off, o_off, fold_off;  // bytes, and where in them
    bool umma;
};

int check_shape(const kvb_shape& s, int q_type, int num_tokens, int max_new, int max_len, int kernel) {
    if (s.batch < 0 || s.num_heads <= 0 || s.num_kv_heads <= 0) return invalid("bad shape");
    if (s.head_dim != 64 && s.head_dim != 128) return invalid("head_dim must be 64 or 128");
    if (s.num_heads % s.num_kv_heads != 0) return invalid("H % Hkv != 0");
    if (s.num_heads / s.num_kv_heads > 64) return invalid("more than 64 query heads per KV head");
    if (s.num_heads > 65536) return invalid("more than 65536 query heads");
    if (q_type != KVB_F32 && q_type != KVB_F16) return invalid("q and out must be f32 or f16");
    if (num_tokens < 0 || max_new < 0 || max_len < 0) return invalid("num_tokens, max_new or max_len < 0");
    if (s.batch > 0 && num_tokens > 0 && max_new < 1) return invalid("max_new must be at least 1");
    if (kernel != KVB_KERNEL_AUTO && kernel != KVB_KERNEL_SIMT && kernel != KVB_KERNEL_UMMA)
        return invalid("unknown kernel");
    return KVB_OK;
}

// The kernel, its units and how many parts the keys are split into. One CTA takes a unit; a call whose
// units leave SMs idle splits the keys of each into parts, merged by a second kernel.
int geometry(Attend& a) {
    int sms = 0;
    if (int rc = kvb_device_sms(&sms)) return rc;
    ChunkParams& p = a.p;
    const kvb_shape& s = a.s;
    p.max_new = std::min(p.max_new, p.T);  // no sequence has more rows than the step, whatever the bound
    p.B = s.batch;
    p.H = s.num_heads;
    p.Hkv = s.num_kv_heads;
    p.G = s.num_heads / s.num_kv_heads;
    p.q_scale = 1.4426950408889634f / std::sqrt(float(s.head_dim));
    // (the tensor maps of fp16 pages number the pool's rows with 31 bits)
    a.umma = a.kernel != KVB_KERNEL_SIMT &&
             kvb_chunk_umma_supported(a.q_type, a.kv_type, a.paged, s.head_dim, p.page, p.G) &&
             (!a.paged || a.kv_type == KVB_I8 || p.num_blocks <= 0x7fffffffll / ((long long)p.Hkv * p.page));
    if (a.kernel == KVB_KERNEL_UMMA && !a.umma)
        return invalid("the requested tensor-core kernel does not support this shape, page size or dtype");
    p.tile_tokens = (a.umma ? 128 : KVB_SIMT_ROWS) / p.G;
    p.unit_tokens = a.umma ? 2 * p.tile_tokens : p.tile_tokens;
    p.blocks_of_new = (std::max(p.max_new, 1) + p.unit_tokens - 1) / p.unit_tokens;
    const long long base = (long long)p.blocks_of_new * p.B * p.Hkv;
    const int64_t head = 256, D = s.head_dim;
    a.workspace = head;
    p.splits = 1;
    if (a.umma) {
        // CTAs that share the work: an SM each, no more than parts of 512 keys of the longest sequences
        const long long most = base * std::max<long long>(1, ((long long)p.max_len + 511) / 512);
        p.ctas = (int)std::min<long long>(most, sms);
        const int fold = a.q_type == KVB_F32 ? KVB_CHUNK_FOLD_F32 : KVB_CHUNK_FOLD_F16;
        a.pieces_off = a.workspace;
        a.ml_off = (int64_t)kvb_align_up(a.pieces_off + sizeof(ChunkPiece) * p.ctas, 256);
        a.o_off = a.ml_off + (int64_t)sizeof(float2) * p.ctas * 2 * 256;
        a.fold_off = a.o_off + 4 * D * p.ctas * 2 * 256;
        a.workspace = a.fold_off + (p.max_len > fold * 128 ? 4 * D * p.ctas * 256 : 0);
        return KVB_OK;
    }
    const long long slots = 2ll * sms, least = 128;  // CTAs that run at once, keys worth a part
    if (base < slots)
        p.splits = (int)std::max<long long>(1, std::min(slots / std::max<long long>(base, 1), p.max_len / least));
    p.units = base * p.splits;
    if (p.units >= (1ll << 31)) return invalid("more than 2^31 work units");
    a.ml_off = head;
    a.o_off = (int64_t)kvb_align_up(head + sizeof(float2) * (size_t)p.splits * p.T * p.H, 256);
    if (p.splits > 1) a.workspace = a.o_off + 4 * D * p.splits * p.T * p.H;
    return KVB_OK;
}

// Tensor maps of what the tcgen05 kernel loads in tiles: fp16 queries as (dim, head, token), boxes of the
// group's heads by a tile's tokens; fp16 pages as (dim, pool row); packed keys and values as (dim, head,
// token). Boxes are 64 values (128 bytes) wide.
int tensor_maps(const Attend& a, CUtensorMap* tq, CUtensorMap* tk, CUtensorMap* tv) {
    const ChunkParams& p = a.p;
    const unsigned long long D = (unsigned long long)a.s.head_dim;
    std::memset(tq, 0, sizeof *tq);
    std::memset(tk, 0, sizeof *tk);
    std::memset(tv, 0, sizeof *tv);
    bool ok = true;
    auto packed = [&](CUtensorMap* m, const void* base, int heads, int64_t stride, unsigned bh, unsigned bt) {
        const unsigned long long dims[3] = {D, (unsigned long long)heads, (unsigned long long)p.T};
        const unsigned long long strides[2] = {2 * D, p.T > 1 ? 2ull * stride : 2 * D * heads};
        const unsigned box[3] = {64, bh, bt};
        ok = ok && kvb_encode_tile_map(m, base, 2, 3, dims, strides, box);
    };
    if (a.q_type == KVB_F16) packed(tq, p.q, p.H, p.q_stride, (unsigned)p.G, (unsigned)p.tile_tokens);
    if (!a.paged) {
        packed(tk, p.k, p.Hkv, p.k_stride, 1, 128);
        packed(tv, p.v, p.Hkv, p.v_stride, 1, 128);
    } else if (a.kv_type == KVB_F16) {
        const unsigned long long dims[2] = {D, (unsigned long long)p.num_blocks * p.Hkv * p.page};
        const unsigned long long strides[1] = {2 * D};
        const unsigned box[2] = {64, (unsigned)std::min(p.page, 128)};
        ok = ok && kvb_encode_tile_map(tk, p.k, 2, 2, dims, strides, box) &&
             kvb_encode_tile_map(tv, p.v, 2, 2, dims, strides, box);
    }
    return ok ? KVB_OK : kvb_fail(KVB_ERR_DEVICE, "cuTensorMapEncodeTiled failed");
}

int run(Attend& a, void* workspace, size_t workspace_bytes, void* stream) {
    ChunkParams& p = a.p;
    if (a.s.batch == 0 || p.T == 0) return KVB_OK;
    if (int rc = geometry(a)) return rc;
    if (!workspace || !aligned32(workspace) || workspace_bytes < (size_t)a.workspace)
        return invalid("workspace null, not 32-byte aligned or too small");
    int sms = 0;
    if (int rc = kvb_device_sms(&sms)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    p.pieces = reinterpret_cast<ChunkPiece*>(ws + a.pieces_off);
    p.part_ml = reinterpret_cast<float2*>(ws + a.ml_off);
    p.part_o = reinterpret_cast<float*>(ws + a.o_off);
    p.fold = reinterpret_cast<float*>(ws + a.fold_off);
    cudaError_t e;
    if (a.umma) {
        CUtensorMap tq, tk, tv;
        if (int rc = tensor_maps(a, &tq, &tk, &tv)) return rc;
        e = kvb_launch_chunk_umma(p, a.q_type, a.kv_type, a.s.head_dim, &tq, &tk, &tv, st);
        if (e == cudaSuccess && p.ctas > 1) e = kvb_launch_chunk_join(p, a.q_type, a.s.head_dim, st);
        return launched(e);
    }
    e = kvb_launch_chunk_simt(p, a.q_type, a.kv_type, a.s.head_dim, st);
    if (e == cudaSuccess && p.splits > 1) e = kvb_launch_chunk_merge(p, a.q_type, a.s.head_dim, sms, st);
    return launched(e);
}

int chunk_attend(const kvb_chunk_args* c, Attend& a) {
    if (!c) return invalid("null arguments");
    const kvb_shape& s = c->shape;
    if (int rc = check_shape(s, c->q_type, c->num_tokens, c->max_new, c->max_len, c->kernel)) return rc;
    if (c->kv_type < KVB_F32 || c->kv_type > KVB_I8) return invalid("unknown kv_type");
    if (c->page_size <= 0 || c->max_blocks < 0) return invalid("page_size <= 0 or max_blocks < 0");
    a = Attend{};
    a.s = s;
    a.q_type = c->q_type;
    a.kv_type = c->kv_type;
    a.kernel = c->kernel;
    a.paged = true;
    ChunkParams& p = a.p;
    p.T = c->num_tokens;
    p.q = c->q;
    p.out = c->out;
    p.k = c->k;
    p.v = c->v;
    p.q_stride = c->q_stride;
    p.k_scale = c->k_scale;
    p.v_scale = c->v_scale;
    p.block_table = c->block_table;
    p.total_lens = c->total_lens;
    p.cu = c->cu_new;
    p.error_flag = c->error_word;
    p.num_blocks = c->num_blocks;
    p.page = c->page_size;
    p.max_blocks = c->max_blocks;
    p.max_new = c->max_new;
    p.max_len = c->max_len;
    if (s.batch == 0 || c->num_tokens == 0) return KVB_OK;
    if (int rc = check_rows(c->q, c->q_stride, (int64_t)s.num_heads * s.head_dim, elem_size(c->q_type), c->num_tokens))
        return rc;
    if (!c->k || !c->v || !c->block_table || !c->total_lens || !c->cu_new || !c->out || !c->error_word)
        return invalid("null device pointer");
    if (c->kv_type == KVB_I8 && (!c->k_scale || !c->v_scale)) return invalid("i8 cache without scales");
    if (!aligned32(c->out) || !aligned16(c->k) || !aligned16(c->v))
        return invalid("out must be 32-byte, k and v 16-byte aligned");
    if (c->num_blocks <= 0) return invalid("num_blocks must be > 0");
    return KVB_OK;
}

int prompt_attend(const kvb_prompt_args* c, Attend& a) {
    if (!c) return invalid("null arguments");
    const kvb_shape& s = c->shape;
    if (int rc = check_shape(s, c->type, c->num_tokens, c->max_len, c->max_len, c->kernel)) return rc;
    a = Attend{};
    a.s = s;
    a.q_type = a.kv_type = c->type;
    a.kernel = c->kernel;
    a.paged = false;
    ChunkParams& p = a.p;
    p.T = c->num_tokens;
    p.q = c->q;
    p.out = c->out;
    p.k = c->k;
    p.v = c->v;
    p.q_stride = c->q_stride;
    p.k_stride = c->k_stride;
    p.v_stride = c->v_stride;
    p.cu = c->cu_lens;
    p.error_flag = c->error_word;
    p.page = 1;
    p.max_new = p.max_len = c->max_len;
    if (s.batch == 0 || c->num_tokens == 0) return KVB_OK;
    const int es = elem_size(c->type);
    const int64_t kv_row = (int64_t)s.num_kv_heads * s.head_dim;
    if (int rc = check_rows(c->q, c->q_stride, (int64_t)s.num_heads * s.head_dim, es, c->num_tokens)) return rc;
    if (int rc = check_rows(c->k, c->k_stride, kv_row, es, c->num_tokens)) return rc;
    if (int rc = check_rows(c->v, c->v_stride, kv_row, es, c->num_tokens)) return rc;
    if (!c->cu_lens || !c->out || !c->error_word) return invalid("null device pointer");
    if (!aligned32(c->out)) return invalid("out must be 32-byte aligned");
    return KVB_OK;
}

int workspace_of(Attend& a, size_t* bytes) {
    if (!bytes) return invalid("null bytes");
    a.workspace = 256;
    if (a.s.batch > 0 && a.p.T > 0)
        if (int rc = geometry(a)) return rc;
    *bytes = (size_t)a.workspace;
    return KVB_OK;
}

}  // namespace

extern "C" {

int kvb_step_plan(const kvb_step_plan_args* a, void* stream) {
    if (!a) return invalid("null arguments");
    if (a->batch < 0 || a->page_size <= 0 || a->max_blocks < 0 || a->num_tokens < 0)
        return invalid("batch, max_blocks or num_tokens < 0 or page_size <= 0");
    if (a->ring_size < 0 || a->num_blocks <= 0) return invalid("ring_size < 0 or num_blocks <= 0");
    if (!a->ring_pos || !a->ring_out || !a->cu_new || (a->ring_size > 0 && !a->ring))
        return invalid("null device pointer");
    if (a->batch > 0 && (!a->seq_lens || !a->new_lens || !a->total_lens)) return invalid("null device pointer");
    if (a->batch > 0 && a->max_blocks > 0 && !a->block_table) return invalid("null block_table");
    if (a->num_tokens > 0 && !a->slot_map) return invalid("null slot_map");
    // CTAs read the inputs at different times, so an output written over one would be read half new
    const size_t B = (size_t)a->batch, T = (size_t)a->num_tokens;
    const void* in[] = {a->seq_lens, a->new_lens, a->ring, a->ring_pos};
    const size_t nin[] = {4 * B, 4 * B, 4 * (size_t)a->ring_size, 16};
    const void* out[] = {a->block_table, a->ring_out, a->total_lens, a->cu_new, a->slot_map, a->positions};
    const size_t nout[] = {4 * B * (size_t)a->max_blocks, 16, 4 * B, 4 * (B + 1), 8 * T, 4 * T};
    for (int i = 0; i < 6; ++i) {
        for (int j = 0; j < 4; ++j)
            if (overlap(out[i], nout[i], in[j], nin[j])) return invalid("an output overlaps an input");
        for (int j = 0; j < i; ++j)
            if (overlap(out[i], nout[i], out[j], nout[j])) return invalid("two outputs overlap");
    }
    PlanParams p;
    p.seq_lens = a->seq_lens;
    p.new_lens = a->new_lens;
    p.block_table = a->block_table;
    p.ring = a->ring;
    p.ring_pos = reinterpret_cast<const long long*>(a->ring_pos);
    p.ring_out = reinterpret_cast<long long*>(a->ring_out);
    p.total_lens = a->total_lens;
    p.cu_new = a->cu_new;
    p.slot_map = reinterpret_cast<long long*>(a->slot_map);
    p.positions = a->positions;
    p.error_flag = a->error_word;
    p.ring_size = a->ring_size;
    p.num_blocks = a->num_blocks;
    p.B = a->batch;
    p.page = a->page_size;
    p.max_blocks = a->max_blocks;
    p.num_tokens = a->num_tokens;
    p.div_page = kvb_div_make((uint32_t)a->page_size);
    int sms = 0;
    if (int rc = kvb_device_sms(&sms)) return rc;
    return launched(kvb_launch_step_plan(p, sms, static_cast<cudaStream_t>(stream)));
}

int kvb_paged_append(const kvb_append_args* a, void* stream) {
    if (!a) return invalid("null arguments");
    const kvb_shape& s = a->shape;
    if (a->src_type != KVB_F32 && a->src_type != KVB_F16) return invalid("rows must be f32 or f16");
    if (a->kv_type < KVB_F32 || a->kv_type > KVB_I8) return invalid("unknown kv_type");
    if (a->kv_type == KVB_F32 && a->src_type != KVB_F32) return invalid("an f32 pool takes f32 rows");
    if (s.batch < 0) return invalid("batch < 0");
    if (s.num_kv_heads < 1 || s.num_kv_heads > 32767) return invalid("num_kv_heads must be in [1, 32767]");
    if (s.head_dim < 8 || s.head_dim % 8 || s.head_dim > 32768)
        return invalid("head_dim must be a multiple of 8 in [8, 32768]");
    if (a->page_size <= 0 || a->max_blocks < 0 || a->num_tokens < 0)
        return invalid("page_size <= 0, max_blocks < 0 or num_tokens < 0");
    if ((int64_t)a->page_size * s.head_dim >= (1ll << 31)) return invalid("a page of one head has 2^31 or more values");
    if (a->num_blocks <= 0) return invalid("num_blocks must be > 0");
    if (a->num_tokens == 0) return KVB_OK;
    const int64_t row = (int64_t)s.num_kv_heads * s.head_dim;
    if (int rc = check_rows(a->k, a->k_stride, row, elem_size(a->src_type), a->num_tokens)) return rc;
    if (int rc = check_rows(a->v, a->v_stride, row, elem_size(a->src_type), a->num_tokens)) return rc;
    if (!a->k_pool || !a->v_pool) return invalid("null device pointer");
    if (!aligned16(a->k_pool) || !aligned16(a->v_pool)) return invalid("pools must be 16-byte aligned");
    const bool i8 = a->kv_type == KVB_I8;
    if (i8 && (!a->k_scale || !a->v_scale)) return invalid("i8 cache without scales");
    if (i8 && (s.batch < 1 || !a->block_table || !a->total_lens || !a->cu_new))
        return invalid("an i8 append takes batch, block_table, total_lens and cu_new");
    if (!i8 && !a->slot_map) return invalid("an f32 or f16 append takes slot_map");
    AppendParams p;
    p.src[0] = a->k;
    p.src[1] = a->v;
    p.stride[0] = a->k_stride;
    p.stride[1] = a->v_stride;
    p.pool[0] = a->k_pool;
    p.pool[1] = a->v_pool;
    p.scale[0] = a->k_scale;
    p.scale[1] = a->v_scale;
    p.slot_map = reinterpret_cast<const long long*>(a->slot_map);
    p.block_table = a->block_table;
    p.total_lens = a->total_lens;
    p.cu_new = a->cu_new;
    p.error_flag = a->error_word;
    p.num_blocks = a->num_blocks;
    p.num_tokens = a->num_tokens;
    p.B = s.batch;
    p.Hkv = s.num_kv_heads;
    p.D = s.head_dim;
    p.page = a->page_size;
    p.max_blocks = a->max_blocks;
    p.div_page = kvb_div_make((uint32_t)a->page_size);
    p.div_row = kvb_div_make((uint32_t)(i8 ? s.head_dim / 4 : s.head_dim * elem_size(a->kv_type) / 16));
    int sms = 0;
    if (int rc = kvb_device_sms(&sms)) return rc;
    return launched(kvb_launch_append(p, a->src_type, a->kv_type, sms, static_cast<cudaStream_t>(stream)));
}

int kvb_paged_chunk_workspace_bytes(const kvb_chunk_args* args, size_t* bytes) {
    Attend a;
    if (int rc = chunk_attend(args, a)) return rc;
    return workspace_of(a, bytes);
}

int kvb_paged_chunk_async(const kvb_chunk_args* args, void* workspace, size_t workspace_bytes, void* stream) {
    Attend a;
    if (int rc = chunk_attend(args, a)) return rc;
    return run(a, workspace, workspace_bytes, stream);
}

int kvb_prompt_workspace_bytes(const kvb_prompt_args* args, size_t* bytes) {
    Attend a;
    if (int rc = prompt_attend(args, a)) return rc;
    return workspace_of(a, bytes);
}

int kvb_prompt_async(const kvb_prompt_args* args, void* workspace, size_t workspace_bytes, void* stream) {
    Attend a;
    if (int rc = prompt_attend(args, a)) return rc;
    return run(a, workspace, workspace_bytes, stream);
}

}  // extern "C"
