// The C ABI's 4-bit floating point calls (h3k_fp4_sizes, h3k_quant_rows_fp4, h3k_dequant_rows_fp4, h3k_gemm_fp4) and the
// attention over packed documents (h3k_attention_packed): checks of the arguments, then the launchers of fp4.cuh and
// attention_packed.cuh.
#include "h3_c.h"

#include "attention_packed.cuh"
#include "common.hpp"
#include "fp4.cuh"

#include <cmath>
#include <functional>
#include <initializer_list>
#include <stdexcept>
#include <string>

namespace h3 {
int run_guarded(const std::function<void()>& f); // capi.cpp: the status codes and message of every entry point
} // namespace h3

namespace {

void need(bool ok, const char* call, const char* what)
{
    if (!ok)
        throw std::invalid_argument(std::string(call) + ": " + what);
}

// Memory that a kernel on the current device may use: not plain host memory, not another device's.
void device_only(const char* call, std::initializer_list<const void*> ptrs)
{
    int current = 0;
    H3_CUDA(cudaGetDevice(&current));
    for (const void* p : ptrs) {
        if (!p)
            continue;
        cudaPointerAttributes a{};
        if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
            cudaGetLastError();
            a.type = cudaMemoryTypeUnregistered;
        }
        need(a.type != cudaMemoryTypeUnregistered && a.devicePointer, call, "a pointer argument is host memory the GPU cannot access");
        need(a.type != cudaMemoryTypeDevice || a.device == current, call, "a pointer argument belongs to another device than the current one");
    }
}

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

h3::Fp4 to_format(const char* call, int32_t format)
{
    need(format == H3K_FP4_MX || format == H3K_FP4_NV, call, "unknown format");
    return h3::Fp4(format);
}

constexpr int32_t kMostDocs = 1 << 30;    // the device's steps past the last one's start are still ints
constexpr int32_t kMostRows = 0x7fffff80; // in whole scale tiles of 128 rows, still an int
constexpr int32_t kMostK = 0x7fffff00;    // in whole stages of 256 values, and a product's rows and columns in whole tiles of 256

void check_rows(const char* call, int32_t rows, int32_t K)
{
    need(rows >= 0, call, "a negative number of rows");
    need(rows <= kMostRows, call, "more than 2^31 - 128 rows");
    need(K > 0 && K % 32 == 0 && K <= kMostK, call, "K must be a positive multiple of 32, at most 2^31 - 256");
}

} // namespace

extern "C" {

int h3k_fp4_sizes(int32_t rows, int32_t K, int32_t format, uint64_t* code_bytes, uint64_t* scale_bytes)
{
    return h3::run_guarded([&] {
        const h3::Fp4 f = to_format("h3k_fp4_sizes", format);
        check_rows("h3k_fp4_sizes", rows, K);
        if (code_bytes)
            *code_bytes = uint64_t(rows) * (K / 2);
        if (scale_bytes)
            *scale_bytes = h3::fp4_scale_bytes(rows, K, f);
    });
}

int h3k_quant_rows_fp4(const void* x, int32_t type, int64_t ldx, int32_t rows, int32_t K, int32_t format, void* codes, void* scales,
                       float* row_scale, void* stream)
{
    return h3::run_guarded([&] {
        const char* call = "h3k_quant_rows_fp4";
        const h3::Fp4 f = to_format(call, format);
        check_rows(call, rows, K);
        need(type >= H3K_BF16 && type <= H3K_F32, call, "unknown element type");
        if (rows == 0)
            return;
        need(x && codes && scales, call, "null argument");
        need((row_scale != nullptr) == (f == h3::Fp4::nv), call, "row_scale is for H3K_FP4_NV, and needed there");
        const int size = type == H3K_F32 ? 4 : 2;
        need(ldx >= 0 && (rows == 1 || ldx * size % 16 == 0), call, "x's rows must be 16 bytes aligned");
        need(aligned(x, 16) && aligned(codes, 16) && aligned(scales, 16) && aligned(row_scale, 4), call, "a pointer is not aligned");
        device_only(call, {x, codes, scales, row_scale});
        h3::quant_rows_fp4(x, h3::Elem(type), ldx, rows, K, f, codes, scales, row_scale, static_cast<cudaStream_t>(stream));
    });
}

int h3k_dequant_rows_fp4(const void* codes, const void* scales, const float* row_scale, int32_t rows, int32_t K, int32_t format, int32_t type,
                         void* out, int64_t ldo, void* stream)
{
    return h3::run_guarded([&] {
        const char* call = "h3k_dequant_rows_fp4";
        const h3::Fp4 f = to_format(call, format);
        check_rows(call, rows, K);
        need(type >= H3K_BF16 && type <= H3K_F32, call, "unknown element type");
        if (rows == 0)
            return;
        need(codes && scales && out, call, "null argument");
        const int size = type == H3K_F32 ? 4 : 2;
        need(rows == 1 || (ldo >= K && ldo * size % 16 == 0), call, "the output's rows must not overlap and be 16 bytes aligned");
        need(aligned(out, 16) && aligned(codes, 16) && aligned(scales, 16) && aligned(row_scale, 4), call, "a pointer is not aligned");
        device_only(call, {codes, scales, row_scale, out});
        h3::dequant_rows_fp4(codes, scales, row_scale, rows, K, f, h3::Elem(type), out, ldo, static_cast<cudaStream_t>(stream));
    });
}

int h3k_gemm_fp4(const void* A, const void* A_scales, const void* B, const void* B_scales, int32_t format, const h3k_gemm_args* a,
                 int32_t epilogue, void* stream)
{
    return h3::run_guarded([&] {
        const char* call = "h3k_gemm_fp4";
        const h3::Fp4 f = to_format(call, format);
        need(a, call, "null argument");
        check_rows(call, a->M, a->K);
        need(a->N > 0 && a->N % 8 == 0, call, "N must be a positive multiple of 8");
        need(a->M <= kMostK && a->N <= kMostK, call, "more than 2^31 - 256 rows or columns");
        need(epilogue >= H3K_EPI_BF16 && epilogue <= H3K_EPI_SWIGLU, call, "unknown epilogue");
        need(a->a_chunks <= 1 && a->a_rows_stride == 0 && (a->lda == 0 || a->lda == a->K) && (a->ldb == 0 || a->ldb == a->K), call,
             "packed rows are contiguous: no chunks or pitches");
        if (a->M == 0)
            return;
        need(A && A_scales && B && B_scales, call, "null argument");
        need(aligned(A, 16) && aligned(A_scales, 16) && aligned(B, 16) && aligned(B_scales, 16) && aligned(a->bias, 16) &&
                 aligned(a->a_scale, 4) && aligned(a->b_scale, 16),
             call, "a pointer is not aligned");
        if (epilogue == H3K_EPI_GATE_RESID) {
            need(a->x && a->mod && a->mod_idx, call, "the gated residual needs x, mod and mod_idx");
            need(a->gate_slot >= 0 && a->gate_slot < 6 && a->dim >= a->N && a->dim % 4 == 0, call, "the gate's slot or the modulation's width");
            need(aligned(a->x, 16) && aligned(a->mod, 16) && (a->M == 1 || (a->ldx >= a->N && a->ldx % 4 == 0)), call,
                 "x's rows must not overlap and be 16 bytes aligned");
        } else {
            need(a->out && aligned(a->out, 16), call, "null or unaligned output");
        }
        if (epilogue == H3K_EPI_BF16 || epilogue == H3K_EPI_F32)
            need(a->M == 1 || (a->ldo >= a->N && a->ldo % (epilogue == H3K_EPI_F32 ? 4 : 8) == 0), call,
                 "the output's rows must not overlap and be 16 bytes aligned");
        if (epilogue == H3K_EPI_SWIGLU) {
            need(a->N % 256 == 0, call, "SwiGLU needs N in 256-row groups");
            need(a->ldo >= a->N / 2 && a->ldo % 8 == 0, call, "the output's rows must not overlap and be 16 bytes aligned");
        }
        if (epilogue == H3K_EPI_QKV) {
            need(a->inner > 0 && a->inner % 256 == 0 && int64_t(a->inner) * 3 == a->N, call, "q/k/v needs N = 3 inner and inner in 256s");
            need(a->heads_per_rank > 0 && (a->inner / 128) % a->heads_per_rank == 0 && a->inner / 128 / a->heads_per_rank <= 8 &&
                     a->rows_local >= a->M,
                 call, "q/k/v head groups or rows");
            need(a->rope && a->qn_w && a->kn_w && aligned(a->rope, 8) && aligned(a->qn_w, 4) && aligned(a->kn_w, 4), call,
                 "q/k/v needs the rotary table and the norms' weights");
        }
        device_only(call, {A, A_scales, B, B_scales, a->out, a->bias, a->x, a->mod, a->mod_idx, a->rope, a->qn_w, a->kn_w, a->a_scale, a->b_scale});
        h3::GemmParams p;
        p.M = a->M, p.N = a->N, p.K = a->K, p.out = a->out, p.ldo = a->ldo, p.bias = a->bias, p.x = a->x, p.ldx = a->ldx;
        p.mod = a->mod, p.mod_idx = a->mod_idx, p.gate_slot = a->gate_slot, p.dim = a->dim, p.rope = a->rope;
        p.qn_w = a->qn_w, p.kn_w = a->kn_w, p.eps = a->eps, p.inner = a->inner, p.heads_per_rank = a->heads_per_rank;
        p.rows_local = a->rows_local, p.a_scale = a->a_scale, p.b_scale = a->b_scale;
        h3::gemm_fp4(A, A_scales, B, B_scales, f, p, h3::Epi(epilogue), static_cast<cudaStream_t>(stream));
    });
}

int h3k_attention_packed(const h3k_packed_args* a, void* stream)
{
    return h3::run_guarded([&] {
        const char* call = "h3k_attention_packed";
        need(a, call, "null argument");
        need(a->type == H3K_BF16 || a->type == H3K_F16, call, "the values are bf16 or f16");
        need(a->head_dim == 64 || a->head_dim == 128, call, "heads have 64 or 128 dims");
        need(a->heads > 0 && a->kv_heads > 0 && a->heads % a->kv_heads == 0 && a->heads / a->kv_heads <= 64 && a->kv_heads <= 65535, call,
             "heads must be a multiple (at most 64) of kv_heads");
        need(a->q_rows >= 0 && a->k_rows >= 0 && a->docs >= 0, call, "a negative number of rows or documents");
        need(a->docs <= kMostDocs, call, "more than 2^30 documents");
        need(a->prefix >= 0 && a->prefix <= a->k_rows, call, "the prefix must lie in the key rows");
        need(a->scale >= 0.f && std::isfinite(a->scale), call, "the scale must be positive (0: 1 / sqrt(head_dim))");
        need(aligned(a->status, 4), call, "a pointer is not aligned");
        if (a->q_rows == 0 || a->docs == 0) {
            if (a->status) {
                device_only(call, {a->status});
                H3_CUDA(cudaMemsetAsync(a->status, 0, sizeof(int32_t), static_cast<cudaStream_t>(stream)));
            }
            return;
        }
        need(a->q && a->out && a->q_start && a->k_start && (a->k_rows == 0 || (a->k && a->v)), call, "null argument");
        need(aligned(a->q, 16) && aligned(a->k, 16) && aligned(a->v, 16) && aligned(a->out, 16) && aligned(a->q_start, 4) && aligned(a->k_start, 4),
             call, "a pointer is not aligned");
        const int64_t q_width = int64_t(a->heads) * a->head_dim, k_width = int64_t(a->kv_heads) * a->head_dim;
        auto rows_ok = [](int rows, int64_t stride, int64_t width) { return rows <= 1 || (stride >= width && stride % 8 == 0); };
        need(rows_ok(a->q_rows, a->q_stride, q_width) && rows_ok(a->q_rows, a->out_stride, q_width) && rows_ok(a->k_rows, a->k_stride, k_width) &&
                 rows_ok(a->k_rows, a->v_stride, k_width),
             call, "rows must not overlap and be 16 bytes aligned");
        device_only(call, {a->q, a->k, a->v, a->out, a->q_start, a->k_start, a->status});
        h3::PackedAttnParams p;
        p.q = a->q, p.k = a->k, p.v = a->v, p.out = a->out, p.q_stride = a->q_stride, p.k_stride = a->k_stride, p.v_stride = a->v_stride;
        p.out_stride = a->out_stride, p.f16 = a->type == H3K_F16, p.heads = a->heads, p.kv_heads = a->kv_heads, p.head_dim = a->head_dim;
        p.q_rows = a->q_rows, p.k_rows = a->k_rows, p.docs = a->docs, p.prefix = a->prefix, p.q_start = a->q_start, p.k_start = a->k_start;
        p.status = a->status;
        p.scale = a->scale > 0.f ? a->scale : 1.f / std::sqrt(float(a->head_dim));
        h3::attention_packed(p, static_cast<cudaStream_t>(stream));
    });
}

} // extern "C"
