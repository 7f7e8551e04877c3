// What the projection GEMMs' kernels (bf16 and int8 in gemm.cu, 4-bit in gemm_fp4.cu) share: the order of the tiles and
// the pieces of their epilogues.
#pragma once
#include "common.hpp"
#include "gemm.cuh"
#include "ptx.cuh"

#include <algorithm>

namespace h3 {

namespace {

constexpr int GROUP_M = 16;

// Destination tensor maps of the TMA-store epilogues. q/k/v: one per rank that owns heads, (dim, q/k/v x head slot,
// row) over that rank's block of this rank's rows, in its receive buffer (fused exchange) or in this rank's send
// layout. SwiGLU: m[0] is the output [M][ldo] (box 64 columns x 128 rows).
struct OutMaps {
    CUtensorMap m[8];
};

__device__ __forceinline__ void epi_bar() { asm volatile("bar.sync 1, 128;" ::: "memory"); } // the 4 epilogue warps

__device__ __forceinline__ void tma_store_3d(const void* tmap, const void* smem_src, int32_t c0, int32_t c1, int32_t c2)
{
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                     reinterpret_cast<uint64_t>(tmap)),
                 "r"(smem_u32(smem_src)), "r"(c0), "r"(c1), "r"(c2)
                 : "memory");
}
__device__ __forceinline__ void tma_store_2d(const void* tmap, const void* smem_src, int32_t c0, int32_t c1)
{
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(reinterpret_cast<uint64_t>(tmap)),
                 "r"(smem_u32(smem_src)), "r"(c0), "r"(c1)
                 : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read0() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait0() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

__device__ __forceinline__ void tile_coords(int tile, int tiles_m, int tiles_n, int& tm, int& tn)
{
    const int group_size = GROUP_M * tiles_n;
    const int g = tile / group_size;
    const int first_m = g * GROUP_M;
    const int gm = min(tiles_m - first_m, GROUP_M);
    const int in_group = tile - g * group_size;
    tm = first_m + in_group % gm;
    tn = in_group / gm;
}

__device__ __forceinline__ float silu(float g) { return g / (1.0f + __expf(-g)); }

__device__ __forceinline__ void store_bf16x32(__nv_bfloat16* dst, const float* v)
{
    uint4* d = reinterpret_cast<uint4*>(dst);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        d[i] = make_uint4(pack_bf16x2(v[8 * i + 0], v[8 * i + 1]), pack_bf16x2(v[8 * i + 2], v[8 * i + 3]),
                          pack_bf16x2(v[8 * i + 4], v[8 * i + 5]), pack_bf16x2(v[8 * i + 6], v[8 * i + 7]));
}

// `rows`: the rows of a q/k/v destination block that the stores may write.
template <Epi EPI>
OutMaps out_maps(const GemmParams& p, int rows)
{
    OutMaps om{};
    if constexpr (EPI == Epi::qkv) {
        // rank r's block of this rank's rows: in r's receive buffer (fused exchange) or in this rank's send layout
        const int P = p.inner / 128 / p.heads_per_rank;
        const uint64_t slots = 3 * uint64_t(p.heads_per_rank);
        const uint64_t odims[3] = {128, slots, uint64_t(rows)};
        const uint64_t ostr[2] = {256, slots * 256};
        const uint32_t obox[3] = {64, 1, 128};
        for (int r = 0; r < P; ++r) {
            const size_t block = size_t(p.peer_out[r] ? p.my_rank : r) * p.rows_local * slots * 128;
            const __nv_bfloat16* base = static_cast<const __nv_bfloat16*>(p.peer_out[r] ? p.peer_out[r] : p.out) + block;
            om.m[r] = make_tmap(CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, base, odims, ostr, obox);
        }
    }
    if constexpr (EPI == Epi::swiglu) {
        const uint64_t odims[2] = {uint64_t(p.N / 2), uint64_t(p.M)};
        const uint64_t ostr[1] = {uint64_t(p.ldo) * 2};
        const uint32_t obox[2] = {64, 128};
        om.m[0] = make_tmap(CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p.out, odims, ostr, obox);
    }
    return om;
}

} // namespace

} // namespace h3
