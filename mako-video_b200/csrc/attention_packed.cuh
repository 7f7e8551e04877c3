// Attention over documents of different lengths packed in one set of rows, with keys that every document sees (a common
// prompt) and kv heads shared by groups of query heads.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace h3 {

struct PackedAttnParams {
    // q: (row, head, dim) at q + row * q_stride + head * head_dim + dim, head < heads; k and v likewise with kv_heads; out as q
    const void* q = nullptr;
    const void* k = nullptr;
    const void* v = nullptr;
    void* out = nullptr;
    int64_t q_stride = 0, k_stride = 0, v_stride = 0, out_stride = 0;
    bool f16 = false; // fp16 values, else bf16
    int heads = 0, kv_heads = 0, head_dim = 128;
    int q_rows = 0, k_rows = 0; // rows of q and out, of k and v
    // Document d: query rows [q_start[d], q_start[d + 1]) see the keys [0, prefix) and [k_start[d], k_start[d + 1]) (device
    // arrays, ascending; a key in both counts once)
    int docs = 0, prefix = 0;
    const int32_t* q_start = nullptr;
    const int32_t* k_start = nullptr;
    float scale = 0.f;
    int32_t* status = nullptr; // 1 where the starts are out of order or out of the rows, else 0 (null: a data error)
};

void attention_packed(const PackedAttnParams& p, cudaStream_t s);

} // namespace h3
