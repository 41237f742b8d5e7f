// Parameters and launchers of the serving-step operators: the step plan, the append into the paged
// cache (kvb_step.cu), and attention of several new tokens per sequence (kvb_chunk_*.cu). Not part
// of the public ABI (that is include/kvb_cuda.h).
#pragma once

#include "kvb_internal.h"

// Helpers of the C ABI's host side (kvb_capi.cu), shared with kvb_step_capi.cu.
int kvb_fail(int code, const char* msg);
int kvb_device_sms(int* num_sms);
// Encodes a tiled tensor map of fp16 (or bytes) with the 128-byte swizzle; rank 2 or 3, strides in
// bytes of dimensions 1.. ; false when the driver refuses it.
bool kvb_encode_tile_map(void* map, const void* base, int elem_size, int rank, const unsigned long long* dims,
                         const unsigned long long* strides, const unsigned* box);

struct PlanParams {
    const int* seq_lens;      // [B]
    const int* new_lens;      // [B]
    int* block_table;         // [B][max_blocks]
    const int* ring;          // [ring_size]
    const long long* ring_pos;  // [2] head, tail
    long long* ring_out;      // [2]
    int* total_lens;          // [B]
    int* cu_new;              // [B + 1]
    long long* slot_map;      // [num_tokens]
    int* positions;           // [num_tokens] or null
    unsigned* error_flag;     // or null
    long long ring_size, num_blocks;
    int B, page, max_blocks, num_tokens;
    KvbDiv div_page;
};
cudaError_t kvb_launch_step_plan(const PlanParams& p, int num_sms, cudaStream_t stream);

struct AppendParams {
    const void* src[2];       // k, v: [num_tokens][Hkv][D], rows of a token contiguous
    long long stride[2];      // elements between tokens
    void* pool[2];            // [num_blocks][Hkv][page][D]
    float* scale[2];          // int8: [num_blocks][Hkv]
    const long long* slot_map;  // fp32, fp16 pools
    const int* block_table;   // int8: [B][max_blocks]
    const int* total_lens;    // int8: [B]
    const int* cu_new;        // int8: [B + 1]
    unsigned* error_flag;     // or null
    long long num_blocks;
    int num_tokens, B, Hkv, D, page, max_blocks;
    KvbDiv div_page, div_row;  // page; pieces of a row (16 pool bytes; int8: four values)
};
cudaError_t kvb_launch_append(const AppendParams& p, int src_type, int kv_type, int num_sms, cudaStream_t stream);
