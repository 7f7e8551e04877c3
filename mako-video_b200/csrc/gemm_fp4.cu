// The projection GEMM on microscaled 4-bit rows (layouts in fp4.cuh): tcgen05.mma kind::mxf4 / kind::mxf4nvf4 with the
// block scales in TMEM, fp32 accumulation, the row scales and the step's epilogues on the way out.
//
// One CTA per SM: warp 0 loads (TMA tiles of 128 bytes = 256 values of K, 128-byte swizzled, and the scale tiles as they lie),
// warp 1 issues, warps 2..9 are the epilogue. Per stage the issuer copies the stage's scale tiles from shared memory into
// TMEM (tcgen05.cp, in order before the MMAs that read them) and runs four MMAs of K = 64 and 128 rows x 256 columns per SM.
// The issue itself is what a stage's 12 copies and 4 MMAs in 512 clocks strain: descriptors are made once a stage and the
// warp stays converged (one lane chosen by elect.sync), which took the main loop of 33024 x 15360 x 5120 from 1.68 ms to
// 0.93 (before the pairs).
//
// Three forms:
//   pair   (more than 128 rows, or few tiles) the two CTAs of a cluster share a tile of 256 x 256: each loads its 128 rows of A and half of
//          B's, the first CTA issues for both (cta_group::2). A stage is 38 KB instead of 54 and five fit: at 54 KB in 512
//          clocks an SM's share of the L2 bandwidth, not the tensor core, sets the pace. 33024 x 15360 x 5120 takes 1.03 ms
//          (5.0 PFLOP/s; tensor pipe 77% at the 1.45 GHz that the power limit leaves) against 1.26 in single CTAs, about
//          0.13 of it the output's stores. The second CTA's loads complete on the first one's barriers; its thread
//          telling the first by a remote arrival a stage took 1.5 ms.
//   tiles  (at most 128 rows, more tiles of 128 x 256 than half the SMs) a CTA walks such tiles: 1 row of 27648 columns and
//          K = 5120 in 21.6 us against 28.0 by pairs, whose second CTA would have no rows
//   split  (fewer such tiles, of few rows or long K: the rule is in launch()) the K of a tile is split over the CTAs of a
//          cluster; they leave their sums in shared memory and each finishes a share of the tile from all of them, in order
//
// TMEM: the accumulator's 256 columns, then the scales of every stage of the ring (48 columns each for nv), so that a stage's
// `empty` barrier covers its scales too; a second accumulator would leave none of the 512 for them. The epilogue's eight
// warps take a finished accumulator into registers at once (128 columns a thread), and the next tile's MMAs start while
// they do the arithmetic and the stores.
#include "common.hpp"
#include "fp4.cuh"
#include "gemm_tiles.cuh"
#include "ptx.cuh"

#include <algorithm>
#include <type_traits>

namespace h3 {

namespace {

constexpr int BM = 128, BN = 256;
constexpr int KSTAGE = 256;          // values of K per stage: 128 bytes of codes a row
constexpr int A_BYTES = BM * 128;
constexpr int EPI_WARPS = 8;
constexpr int NUM_THREADS = 64 + 32 * EPI_WARPS;
constexpr int SCALE_COL = BN, SCALE_COLS = 48; // TMEM: the first stage's scales, columns a stage
constexpr int MAX_SPLIT = 8;         // CTAs of a cluster that share a tile's K

enum class Form { tiles, split, pair };

template <Fp4 F, Form W>
struct Fp4Smem {
    static constexpr int STAGES = W == Form::pair ? 5 : 3;
    static constexpr int B_ROWS = W == Form::pair ? BN / 2 : BN; // of a tile, in this CTA
    static constexpr int B_BYTES = B_ROWS * 128;
    // scale tiles of a stage: 4 (nv) or 2 (mx) along K for A's 128 rows and twice as many for B's 256
    static constexpr int KT = KSTAGE / (4 * fp4_block(F));
    static constexpr int SF_BYTES = 3 * KT * 512;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + SF_BYTES;
    // 4 KB an epilogue warp: 32 rows of 128 bytes of output; before that its columns' scales and biases, 2 x 128 floats
    static constexpr int OFF_STAGING = STAGES * STAGE_BYTES;
    static constexpr int OFF_BAR = OFF_STAGING + EPI_WARPS * 4096;
    static constexpr int TOTAL = OFF_BAR + 256 + 1024;
    static_assert(STAGE_BYTES % 1024 == 0 && TOTAL <= 227 * 1024 && BN + STAGES * 48 <= 512);
    static_assert(BM * BN * 4 <= OFF_STAGING); // a split tile's sums, over the ring
};

// A's and B's codes (byte of K, row), and their scale tiles (word of a tile, tile).
struct Fp4Inputs {
    CUtensorMap a, b, a_scales, b_scales;
};

// Destination of the tiles: q/k/v one map per rank that owns heads (dim, q/k/v x head slot, row), else m[0] (column, row).
// Boxes are an epilogue warp's 32 rows of 128 bytes.
template <Epi EPI>
struct Fp4Maps {
    CUtensorMap m[EPI == Epi::qkv ? 8 : 1];
};

// D[tmem] (+)= A[smem] B[smem]^T on e2m1 codes, the block scales in TMEM at sfa and sfb. PAIR: on both CTAs of the pair, each
// with its own rows of A and D, half of B's rows, its scales of A and all of B's.
#define H3_MMA_FP4(GROUP, KIND)                                                                                                   \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"                                                               \
                 "tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),                 \
                 "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)                                                   \
                 : "memory")
template <Fp4 F, bool PAIR>
__device__ __forceinline__ void mma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate)
{
    if constexpr (F == Fp4::nv && PAIR)
        H3_MMA_FP4("2", "mxf4nvf4.block_scale.scale_vec::4X");
    else if constexpr (F == Fp4::nv)
        H3_MMA_FP4("1", "mxf4nvf4.block_scale.scale_vec::4X");
    else if constexpr (PAIR)
        H3_MMA_FP4("2", "mxf4.block_scale.scale_vec::2X");
    else
        H3_MMA_FP4("1", "mxf4.block_scale.scale_vec::2X");
}
#undef H3_MMA_FP4

// Instruction descriptor of the two kinds: e2m1 A and B, both K-major; the scales' type (1: powers of two, 0: e4m3) and
// which pair of the scale bytes of a TMEM word the MMA reads (mx: a word holds two MMAs' scales).
template <Fp4 F, bool PAIR>
__device__ __forceinline__ constexpr uint32_t idesc_fp4(uint32_t pair)
{
    return (pair << 4) | (1u << 7) | (1u << 10) | (uint32_t(BN >> 3) << 17) | (uint32_t(F == Fp4::mx) << 23) |
           (uint32_t((PAIR ? 2 * BM : BM) >> 7) << 27) | (pair << 29);
}

// The scale copies and MMAs of one stage: `tiles` scale tiles along K and `steps` MMAs (constants in full stages, so that
// the loops unroll). Scale tile k of A goes to columns tsf + 12 k, of B's two row halves to the next four and four.
template <Fp4 F, bool PAIR>
__device__ __forceinline__ void issue_stage(uint32_t d, uint64_t ad, uint64_t bd, uint64_t fd, uint32_t tsf, int tiles, int steps, bool fresh)
{
    constexpr int KT = Fp4Smem<F, Form::tiles>::KT;
#pragma unroll
    for (int k = 0; k < tiles; ++k)
#pragma unroll
        for (int x = 0; x < 3; ++x) {
            // one tile, 32 rows of 16 bytes, into four columns of 32 lanes, repeated for the four lane quarters
            const uint64_t from = fd + (x * KT + k) * (512 >> 4);
            if constexpr (PAIR)
                asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tsf + k * 12 + x * 4), "l"(from) : "memory");
            else
                asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tsf + k * 12 + x * 4), "l"(from) : "memory");
        }
#pragma unroll
    for (int k = 0; k < steps; ++k) {
        const uint32_t sf = tsf + (F == Fp4::nv ? k : k / 2) * 12;
        mma_fp4<F, PAIR>(d, ad + k * (32 >> 4), bd + k * (32 >> 4), idesc_fp4<F, PAIR>(F == Fp4::nv ? 0 : (k & 1) * 2), sf, sf + 4, !fresh || k > 0);
    }
}

// Arrive on `bar` (of both CTAs of a pair) once every tcgen05 operation this thread issued before has completed.
template <bool PAIR>
__device__ __forceinline__ void commit(uint64_t* bar)
{
    if constexpr (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                     "h"(uint16_t(3))
                     : "memory");
    else
        mma_commit(bar);
}

// Arrives on the barrier at the same place in CTA `rank` of the cluster. (What it orders is tensor memory, by the tcgen05
// fences around it.)
__device__ __forceinline__ void arrive_cluster(uint64_t* bar, uint32_t rank)
{
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, %1;\n\tmbarrier.arrive.shared::cluster.b64 _, [a];\n\t}" ::"r"(smem_u32(bar)),
                 "r"(rank)
                 : "memory");
}

// A TMA tile into this CTA's shared memory that completes on `bar`, a shared::cluster address: a pair's first CTA counts the
// loads of both.
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const void* tmap, uint32_t bar, int32_t c0, int32_t c1)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];" ::"r"(
                     smem_u32(dst)),
                 "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(c0), "r"(c1)
                 : "memory");
}

// mbar_wait for a barrier that the cluster's other CTA arrives on.
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity)
{
    auto done = [&] {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, 1000000;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok)
                     : "r"(smem_u32(bar)), "r"(parity)
                     : "memory");
        return ok != 0;
    };
    if (done())
        return true;
    const long long t0 = clock64();
    for (uint32_t i = 1;; ++i) {
        if (done())
            return true;
        if (clock64() - t0 > 4000000000ll) {
            record_error(kErrWaitTimeout);
            return false;
        }
        if ((i & 255) == 0 && *(volatile uint32_t*)&g_device_error != 0)
            return false;
    }
}

template <bool PAIR>
__device__ __forceinline__ void tmem_get(uint32_t* slot)
{
    if constexpr (PAIR) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        tmem_alloc(slot, 512);
        tmem_relinquish();
    }
}
template <bool PAIR>
__device__ __forceinline__ void tmem_free(uint32_t tmem)
{
    if constexpr (PAIR)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    else
        tmem_dealloc(tmem, 512);
}

__device__ __forceinline__ void tma_reduce_add_2d(const void* tmap, const void* smem_src, int32_t c0, int32_t c1)
{
    asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                     reinterpret_cast<uint64_t>(tmap)),
                 "r"(smem_u32(smem_src)), "r"(c0), "r"(c1)
                 : "memory");
}

__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr, uint32_t rank)
{
    float4 v;
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\tld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n\t}"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr), "r"(rank)
                 : "memory");
    return v;
}

// silu: g / (1 + e^-g), by the approximate reciprocal (1 ulp), which the rounding to bf16 hides. Both sides are a sixteenth, since the
// reciprocal of a number above 2^126 would be flushed to 0: the result is 0 only where e^-g / 16 is (g below -90.1,
// where silu is below 2^-123). As a division in full precision, 512 x 27648 x 5120 takes 57 us instead of 33.
__device__ __forceinline__ float silu_approx(float g)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(0.0625f + ex2_approx(fmaf(g, -1.4426950408889634f, -4.0f))));
    return g * 0.0625f * r;
}

// First column, within the tile, of the chunk c (of four of 32 columns) that an epilogue thread of a half holds: the SwiGLU
// pairs gate column j with value column 128 + j, so a thread takes 64 of both; else 128 columns in a row.
template <Epi EPI>
__device__ __forceinline__ int chunk_col(int half, int c)
{
    return EPI == Epi::swiglu ? half * 64 + (c >> 1) * 128 + (c & 1) * 32 : half * 128 + c * 32;
}

// Piece `i` (16 bytes) of this lane's 128-byte row of the warp's staging buffer, swizzled as the tensor map has it.
__device__ __forceinline__ void stage_piece(uint8_t* buf, int i, uint4 v) { *reinterpret_cast<uint4*>(buf + lane_id() * 128 + ((i ^ (lane_id() & 7)) << 4)) = v; }
__device__ __forceinline__ uint4 pack8(const float* v)
{
    return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

// The epilogue of this warp's 32 rows x 128 columns: takes the accumulator (release() once it is in registers), then 4 KB
// of finished output at a time through the warp's staging buffer, stored by TMA (which clips rows past M and columns past
// N). The buffer holds the columns' row scales of B and their biases first.
template <Epi EPI, class Release>
__device__ __forceinline__ void epilogue_fp4(const GemmParams& p, uint32_t taddr, int m0, int n0, int half, uint8_t* buf, const Fp4Maps<EPI>& om,
                                             Release&& release)
{
    const float* cols = reinterpret_cast<const float*>(buf);
    const int gm = m0 + lane_id(); // m0: the warp's first row
    const bool valid = gm < p.M;
    const float a_scale = p.a_scale && valid ? __ldg(p.a_scale + gm) : 1.0f;
    float v[128];
    {
        uint32_t r[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c)
            tmem_ld32(taddr + chunk_col<EPI>(half, c), r[c]);
        tmem_wait_ld();
        release();
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
                v[c * 32 + i] = __uint_as_float(r[c][i]);
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        const float4 s = reinterpret_cast<const float4*>(cols)[i], b = reinterpret_cast<const float4*>(cols + 128)[i];
        v[4 * i] = fmaf(v[4 * i], a_scale * s.x, b.x), v[4 * i + 1] = fmaf(v[4 * i + 1], a_scale * s.y, b.y);
        v[4 * i + 2] = fmaf(v[4 * i + 2], a_scale * s.z, b.z), v[4 * i + 3] = fmaf(v[4 * i + 3], a_scale * s.w, b.w);
    }
    // ready(): the staging buffer's last store has read it; send(): the warp's rows are in it
    auto ready = [&] {
        if (lane_id() == 0)
            bulk_wait_read0();
        __syncwarp();
    };
    auto send = [&](auto&& store) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane_id() == 0 && m0 < p.M) {
            store();
            bulk_commit();
        }
    };

    if constexpr (EPI == Epi::qkv) {
        const int col = n0 + half * 128;
        const int sec = n0 / p.inner;
        if (sec < 2) {
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < 128; ++j)
                ss += v[j] * v[j];
            const float rinv = rsqrtf(ss * (1.0f / 128.0f) + p.eps);
            const float* w = sec == 0 ? p.qn_w : p.kn_w;
#pragma unroll
            for (int j = 0; j < 128; ++j)
                v[j] = v[j] * rinv * __ldg(w + j);
            const float2* cs = reinterpret_cast<const float2*>(p.rope) + size_t(valid ? gm : p.M - 1) * 48;
#pragma unroll
            for (int j = 0; j < 48; ++j) {
                const float2 t = __ldg(cs + j);
                const float a = v[j], b = v[j + 48];
                v[j] = a * t.x - b * t.y;
                v[j + 48] = b * t.x + a * t.y;
            }
        }
        const int head = (col % p.inner) / 128;
        const int rank = head / p.heads_per_rank, slot = sec * p.heads_per_rank + head % p.heads_per_rank;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            ready();
#pragma unroll
            for (int i = 0; i < 8; ++i)
                stage_piece(buf, i, pack8(v + h * 64 + i * 8));
            send([&] { tma_store_3d(&om.m[rank], buf, h * 64, slot, m0); });
        }
    } else if constexpr (EPI == Epi::swiglu) {
#pragma unroll
        for (int j = 0; j < 64; ++j)
            v[j] = silu_approx(v[j]) * v[64 + j];
        ready();
#pragma unroll
        for (int i = 0; i < 8; ++i)
            stage_piece(buf, i, pack8(v + i * 8));
        send([&] { tma_store_2d(&om.m[0], buf, n0 / 2 + half * 64, m0); });
    } else if constexpr (EPI == Epi::bf16) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            ready();
#pragma unroll
            for (int i = 0; i < 8; ++i)
                stage_piece(buf, i, pack8(v + h * 64 + i * 8));
            const int col = n0 + half * 128 + h * 64;
            send([&] {
                if (col < p.N)
                    tma_store_2d(&om.m[0], buf, col, m0);
            });
        }
    } else {
        // f32 as it is; the gated residual adds gate * v to x where x lies (one fp32 addition per value, by the TMA reduction)
        if constexpr (EPI == Epi::gate_resid) {
            const float4* g4 = reinterpret_cast<const float4*>(p.mod + (size_t(valid ? p.mod_idx[gm] : 0) * 6 + p.gate_slot) * p.dim + n0 + half * 128);
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (n0 + half * 128 + 4 * i < p.N) {
                    const float4 g = __ldg(g4 + i);
                    v[4 * i] *= g.x, v[4 * i + 1] *= g.y, v[4 * i + 2] *= g.z, v[4 * i + 3] *= g.w;
                }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            ready();
#pragma unroll
            for (int i = 0; i < 8; ++i)
                stage_piece(buf, i, *reinterpret_cast<const uint4*>(v + c * 32 + i * 4));
            const int col = n0 + half * 128 + c * 32;
            send([&] {
                if (col < p.N) {
                    if constexpr (EPI == Epi::f32)
                        tma_store_2d(&om.m[0], buf, col, m0);
                    else
                        tma_reduce_add_2d(&om.m[0], buf, col, m0);
                }
            });
        }
    }
}

// Four columns from `col` of row gm of a split tile: the parts' sums (s, and u for the SwiGLU's values at column col + 128)
// through the epilogue, straight to the output.
template <Epi EPI>
__device__ __forceinline__ void finish4(const GemmParams& p, float4 s, float4 u, int gm, int col)
{
    const float a = p.a_scale ? __ldg(p.a_scale + gm) : 1.f;
    auto scaled = [&](float4 v, int c) {
        const float4 b = p.b_scale ? __ldg(reinterpret_cast<const float4*>(p.b_scale + c)) : make_float4(1.f, 1.f, 1.f, 1.f);
        const float4 d = p.bias ? __ldg(reinterpret_cast<const float4*>(p.bias + c)) : make_float4(0.f, 0.f, 0.f, 0.f);
        return make_float4(fmaf(v.x, a * b.x, d.x), fmaf(v.y, a * b.y, d.y), fmaf(v.z, a * b.z, d.z), fmaf(v.w, a * b.w, d.w));
    };
    float4 v = scaled(s, col);
    if constexpr (EPI == Epi::gate_resid) {
        const float4 g = __ldg(reinterpret_cast<const float4*>(p.mod + (size_t(p.mod_idx[gm]) * 6 + p.gate_slot) * p.dim + col));
        float4* x = reinterpret_cast<float4*>(p.x + size_t(gm) * p.ldx + col);
        float4 o = *x;
        o.x = __fadd_rn(o.x, v.x * g.x), o.y = __fadd_rn(o.y, v.y * g.y), o.z = __fadd_rn(o.z, v.z * g.z), o.w = __fadd_rn(o.w, v.w * g.w);
        *x = o;
    } else if constexpr (EPI == Epi::f32) {
        *reinterpret_cast<float4*>(static_cast<float*>(p.out) + size_t(gm) * p.ldo + col) = v;
    } else {
        int at = col;
        if constexpr (EPI == Epi::swiglu) {
            u = scaled(u, col + 128);
            v = make_float4(silu_approx(v.x) * u.x, silu_approx(v.y) * u.y, silu_approx(v.z) * u.z, silu_approx(v.w) * u.w);
            at = (col >> 8) * 128 + (col & 127);
        }
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + size_t(gm) * p.ldo + at) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
    }
}

template <Epi EPI, Fp4 F, Form W>
__global__ void __launch_bounds__(NUM_THREADS, 1)
    gemm_fp4_kernel(const __grid_constant__ Fp4Inputs in, const GemmParams p, const __grid_constant__ Fp4Maps<EPI> om)
{
    using SM = Fp4Smem<F, W>;
    constexpr int KT = SM::KT, STAGES = SM::STAGES;
    constexpr bool SPLIT = W == Form::split, PAIR = W == Form::pair;
    constexpr int TILE_M = PAIR ? 2 * BM : BM;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t* smem = smem_raw + (((raw + 1023) & ~1023u) - raw);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + SM::OFF_BAR);
    uint64_t* full = bars;              // [STAGES] a stage has landed (pair: in both CTAs, counted in the first)
    uint64_t* empty = full + STAGES;    // [STAGES]
    uint64_t* tfull = empty + STAGES;   // the accumulator is complete
    uint64_t* taken = tfull + 1;        // it is in the epilogue's registers (pair: of both CTAs, in the first)
    uint64_t* drain = taken + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);

    const int warp = __shfl_sync(0xffffffffu, warp_id(), 0);
    const int tiles_m = (p.M + TILE_M - 1) / TILE_M, tiles_n = (p.N + BN - 1) / BN;
    const int num_tiles = tiles_m * tiles_n;
    const int scale_tiles = fp4_scale_tiles(p.K, F);
    int first_tile = blockIdx.x, tile_step = gridDim.x;
    int kb0 = 0, kb1 = (p.K + KSTAGE - 1) / KSTAGE; // this CTA's stages of K
    uint32_t split = 1, part = 0;
    if constexpr (SPLIT) {
        asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(split));
        asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(part));
        first_tile = blockIdx.x / split, tile_step = num_tiles;
        const int all = kb1; // every part has a stage: the launch has no more parts than stages
        kb0 = int(part) * all / int(split), kb1 = (int(part) + 1) * all / int(split);
    }
    if constexpr (PAIR) {
        asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(part));
        first_tile = blockIdx.x / 2, tile_step = gridDim.x / 2;
    }

    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        mbar_init(tfull, 1);
        mbar_init(taken, PAIR ? 2 * EPI_WARPS : EPI_WARPS);
        mbar_init(drain, 1);
        fence_barrier_init();
    }
    if (warp == 1)
        tmem_get<PAIR>(tmem_slot);
    tc_fence_before();
    __syncthreads();
    if constexpr (PAIR)
        cluster_sync(); // both CTAs' barriers and TMEM are there
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0 && elect_one_lane()) {
        // ---------------------------------------------------------------------------------------- producer
        uint32_t it = 0;
        bool ok = true;
        for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step) {
            int tm, tn;
            tile_coords(tile, tiles_m, tiles_n, tm, tn);
            const int m_tile = PAIR ? 2 * tm + int(part) : tm; // this CTA's 128 rows (past M in a pair's last tile: zeros)
            for (int kb = kb0; kb < kb1; ++kb, ++it) {
                const int s = it % STAGES;
                if (!(ok = mbar_wait(&empty[s], ((it / STAGES) & 1) ^ 1)))
                    break;
                uint8_t* sa = smem + s * SM::STAGE_BYTES;
                uint8_t* sb = sa + A_BYTES;
                uint8_t* sf = sb + SM::B_BYTES;
                const int b_row = tn * BN + (PAIR ? int(part) * SM::B_ROWS : 0);
                if constexpr (PAIR) {
                    // scale boxes are whole (a tile past the last one of a row range is the next range's, or zeros: not used)
                    if (part == 0)
                        mbar_arrive_expect_tx(&full[s], 2 * SM::STAGE_BYTES);
                    uint32_t bar;
                    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(bar) : "r"(smem_u32(&full[s])));
                    tma_load_2d_pair(sa, &in.a, bar, kb * 128, m_tile * BM);
                    tma_load_2d_pair(sb, &in.b, bar, kb * 128, b_row);
                    tma_load_2d_pair(sf, &in.a_scales, bar, 0, m_tile * scale_tiles + kb * KT);
                    tma_load_2d_pair(sf + KT * 512, &in.b_scales, bar, 0, 2 * tn * scale_tiles + kb * KT);
                    tma_load_2d_pair(sf + 2 * KT * 512, &in.b_scales, bar, 0, (2 * tn + 1) * scale_tiles + kb * KT);
                } else {
                    mbar_arrive_expect_tx(&full[s], SM::STAGE_BYTES);
                    tma_load_2d(sa, &in.a, &full[s], kb * 128, m_tile * BM);
                    tma_load_2d(sb, &in.b, &full[s], kb * 128, b_row);
                    tma_load_2d(sf, &in.a_scales, &full[s], 0, m_tile * scale_tiles + kb * KT);
                    tma_load_2d(sf + KT * 512, &in.b_scales, &full[s], 0, 2 * tn * scale_tiles + kb * KT);
                    tma_load_2d(sf + 2 * KT * 512, &in.b_scales, &full[s], 0, (2 * tn + 1) * scale_tiles + kb * KT);
                }
            }
        }
        // Wait for the loads still in flight to land before the CTA can exit: until the MMAs have read them, or, when a wait gave up and
        // no MMA may follow, for as many times the time that a load takes.
        for (uint32_t j = it >= STAGES ? it - STAGES : 0; j < it; ++j)
            mbar_wait_landed(&empty[j % STAGES], (j / STAGES) & 1, ok ? 4000000000ll : 100000000ll);
    } else if (warp == 1 && (!PAIR || part == 0)) {
        // ------------------------------------------------------------------------------------- MMA issuer
        uint32_t elected;
        asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(elected));
        const uint32_t smem0 = smem_u32(smem);
        uint32_t it = 0, t_local = 0;
        bool ok = true;
        for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step, ++t_local) {
            if (t_local > 0 && !(ok = mbar_wait_cluster(taken, (t_local - 1) & 1)))
                break;
            tc_fence_after();
            for (int kb = kb0; kb < kb1; ++kb, ++it) {
                const int s = it % STAGES;
                if (!(ok = mbar_wait_cluster(&full[s], (it / STAGES) & 1)))
                    break;
                tc_fence_after();
                const uint32_t sa = smem0 + s * SM::STAGE_BYTES, sf = sa + A_BYTES + SM::B_BYTES;
                const uint64_t ad = sdesc_sw128(sa, 16, 1024), bd = sdesc_sw128(sa + A_BYTES, 16, 1024);
                // scale tiles: 8-row groups of 128 bytes, no swizzle
                const uint64_t fd = uint64_t((sf >> 4) & 0x3FFF) | (uint64_t(128 >> 4) << 32) | (uint64_t(1) << 46);
                const uint32_t tsf = tmem + SCALE_COL + s * SCALE_COLS;
                const int left = p.K - kb * KSTAGE;
                if (elected) {
                    if (left >= KSTAGE)
                        issue_stage<F, PAIR>(tmem, ad, bd, fd, tsf, KT, KSTAGE / 64, kb == kb0);
                    else
                        issue_stage<F, PAIR>(tmem, ad, bd, fd, tsf, scale_tiles - kb * KT, (left + 63) / 64, kb == kb0);
                    commit<PAIR>(&empty[s]);
                }
                __syncwarp();
            }
            if (ok && elected)
                commit<PAIR>(tfull);
            __syncwarp();
        }
        // Every MMA this warp issued has completed once `drain` flips.
        if (elected)
            commit<PAIR>(drain);
        __syncwarp();
        mbar_wait_landed(drain, 0);
    } else if (warp >= 2) {
        // ---------------------------------------------------------------------------------------- epilogue
        const int quarter = warp & 3, half = (warp - 2) >> 2; // its 32 TMEM lanes, its half of the columns
        const uint32_t lanes = uint32_t(quarter * 32) << 16;
        if constexpr (SPLIT) {
            // This part's sums, rows below M only: row r's 16-byte piece i at (i ^ (r & 7)), over the ring (its loads have
            // been read by the MMAs that `tfull` follows).
            int tm, tn;
            tile_coords(first_tile, tiles_m, tiles_n, tm, tn);
            const int r = quarter * 32 + lane_id();
            if (mbar_wait(tfull, 0)) {
                tc_fence_after();
                if (tm * BM + quarter * 32 < p.M) {
                    float4* row = reinterpret_cast<float4*>(smem) + r * (BN / 4);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t o[32];
                        tmem_ld32(tmem + lanes + half * 128 + c * 32, o);
                        tmem_wait_ld();
                        if (tm * BM + r < p.M)
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                row[(half * 32 + c * 8 + i) ^ (r & 7)] = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                                                                                     __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
                    }
                }
            }
        } else {
            uint8_t* buf = smem + SM::OFF_STAGING + (warp - 2) * 4096;
            auto release = [&] {
                tc_fence_before();
                __syncwarp();
                if (elect_one_lane()) {
                    if constexpr (PAIR)
                        arrive_cluster(taken, 0);
                    else
                        mbar_arrive(taken);
                }
            };
            uint32_t t_local = 0;
            for (int tile = first_tile; tile < num_tiles; tile += tile_step, ++t_local) {
                int tm, tn;
                tile_coords(tile, tiles_m, tiles_n, tm, tn);
                {
                    // the columns' scales and biases, four a lane, while the MMAs run
                    const int j = lane_id() * 4, col = tn * BN + chunk_col<EPI>(half, j >> 5) + (j & 31);
                    const float4 one = make_float4(1.f, 1.f, 1.f, 1.f), none = make_float4(0.f, 0.f, 0.f, 0.f);
                    float* cols = reinterpret_cast<float*>(buf);
                    if (lane_id() == 0)
                        bulk_wait_read0(); // the tile before has been read from the buffer
                    __syncwarp();
                    reinterpret_cast<float4*>(cols)[lane_id()] = p.b_scale && col < p.N ? __ldg(reinterpret_cast<const float4*>(p.b_scale + col)) : one;
                    reinterpret_cast<float4*>(cols + 128)[lane_id()] = p.bias && col < p.N ? __ldg(reinterpret_cast<const float4*>(p.bias + col)) : none;
                    __syncwarp();
                }
                if (!mbar_wait(tfull, t_local & 1))
                    break;
                tc_fence_after();
                epilogue_fp4<EPI>(p, tmem + lanes, tm * TILE_M + (PAIR ? int(part) * BM : 0) + quarter * 32, tn * BN, half, buf, om, release);
            }
            if (lane_id() == 0)
                bulk_wait0(); // the staged tiles' stores are complete
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) {
        // The closing commit arrives in both CTAs, each of which has to see it before its shared memory may go: that it has
        // arrived in the first says nothing of the second. (Here, after the tiles, so that the wait's bound is not theirs.)
        if (part == 1 && warp == 1)
            mbar_wait_landed(drain, 0);
        cluster_sync(); // no MMA of the pair is under way
    }
    if (warp == 1) {
        tc_fence_after();
        tmem_free<PAIR>(tmem);
    }
    if constexpr (SPLIT) {
        // The tile's rows below M in groups of four columns (SwiGLU: of outputs), dealt out over the cluster's threads.
        cluster_sync();
        int tm, tn;
        tile_coords(first_tile, tiles_m, tiles_n, tm, tn);
        constexpr int GROUPS = EPI == Epi::swiglu ? BN / 8 : BN / 4;
        const int rows = min(BM, p.M - tm * BM);
        for (int i = int(part) * NUM_THREADS + threadIdx.x; i < rows * GROUPS; i += int(split) * NUM_THREADS) {
            const int r = i / GROUPS, g = i % GROUPS, col = tn * BN + g * 4;
            if (col >= p.N)
                continue;
            auto sum = [&](int piece) {
                const uint32_t at = smem_u32(smem) + (r * (BN / 4) + (piece ^ (r & 7))) * 16;
                float4 v[MAX_SPLIT]; // loads under way together
#pragma unroll
                for (uint32_t z = 0; z < MAX_SPLIT; ++z)
                    v[z] = z < split ? ld_cluster4(at, z) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (uint32_t z = 1; z < MAX_SPLIT; ++z)
                    v[0].x += v[z].x, v[0].y += v[z].y, v[0].z += v[z].z, v[0].w += v[z].w;
                return v[0];
            };
            const float4 s = sum(g);
            finish4<EPI>(p, s, EPI == Epi::swiglu ? sum(g + 32) : s, tm * BM + r, col);
        }
        cluster_sync(); // no CTA leaves while another reads its shared memory
    }
}

template <Epi EPI>
Fp4Maps<EPI> output_maps(const GemmParams& p)
{
    Fp4Maps<EPI> om{};
    if constexpr (EPI == Epi::qkv) {
        const int P = p.inner / 128 / p.heads_per_rank;
        const uint64_t slots = 3 * uint64_t(p.heads_per_rank);
        const uint64_t dims[3] = {128, slots, uint64_t(p.M)}, pitch[2] = {256, slots * 256};
        const uint32_t box[3] = {64, 1, 32};
        for (int r = 0; r < P; ++r)
            om.m[r] = make_tmap(CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, static_cast<const __nv_bfloat16*>(p.out) + size_t(r) * p.rows_local * slots * 128, dims,
                                pitch, box);
    } else {
        constexpr bool wide = EPI == Epi::f32 || EPI == Epi::gate_resid;
        const int64_t ld = EPI == Epi::gate_resid ? p.ldx : p.ldo;
        const uint64_t n = EPI == Epi::swiglu ? p.N / 2 : p.N, size = wide ? 4 : 2;
        const uint64_t dims[2] = {n, uint64_t(p.M)}, pitch[1] = {(p.M > 1 ? uint64_t(ld) : (n + 7) / 8 * 8) * size};
        const uint32_t box[2] = {wide ? 32u : 64u, 32};
        om.m[0] = make_tmap(wide ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                            EPI == Epi::gate_resid ? static_cast<const void*>(p.x) : p.out, dims, pitch, box);
    }
    return om;
}

template <Epi EPI, Fp4 F, Form W>
bool launch(const void* A, const void* a_scales, const void* B, const void* b_scales, const GemmParams& p, int tiles, int ctas, cudaStream_t s)
{
    using SM = Fp4Smem<F, W>;
    const uint64_t bytes = uint64_t(p.K) / 2;
    const uint64_t adims[2] = {bytes, uint64_t(p.M)}, bdims[2] = {bytes, uint64_t(p.N)}, pitch[1] = {bytes};
    const uint32_t abox[2] = {128, BM}, bbox[2] = {128, SM::B_ROWS};
    Fp4Inputs in;
    in.a = make_tmap(CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, A, adims, pitch, abox);
    in.b = make_tmap(CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, B, bdims, pitch, bbox);
    const uint64_t scale_tiles = fp4_scale_tiles(p.K, F), spitch[1] = {512};
    const uint64_t asdims[2] = {128, (p.M + 127) / 128 * scale_tiles}, bsdims[2] = {128, (p.N + 127) / 128 * scale_tiles};
    const uint32_t sbox[2] = {128, uint32_t(SM::KT)};
    in.a_scales = make_tmap(CU_TENSOR_MAP_DATA_TYPE_INT32, 2, a_scales, asdims, spitch, sbox, false);
    in.b_scales = make_tmap(CU_TENSOR_MAP_DATA_TYPE_INT32, 2, b_scales, bsdims, spitch, sbox, false);
    Fp4Maps<EPI> om{};
    if constexpr (W != Form::split)
        om = output_maps<EPI>(p);
    static std::atomic<uint64_t> opt_in;
    smem_opt_in(gemm_fp4_kernel<EPI, F, W>, SM::TOTAL, opt_in);
    cudaLaunchConfig_t c{};
    c.blockDim = dim3(NUM_THREADS);
    c.dynamicSmemBytes = SM::TOTAL;
    c.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    c.attrs = at;
    if constexpr (W == Form::pair) {
        c.numAttrs = 1;
        at[0].val.clusterDim.x = 2;
    }
    if constexpr (W == Form::split) {
        int split;
        // the largest cluster of which the device holds one per tile at once, with a stage for every CTA
        c.numAttrs = 1;
        static ClusterLimits limits;
        for (split = std::min({ctas / tiles, MAX_SPLIT, (p.K + KSTAGE - 1) / KSTAGE}); split > 1; --split)
            if (limits.at_once(gemm_fp4_kernel<EPI, F, W>, c, split) >= tiles)
                break;
        // Against pairs of 128 columns a CTA, with which a stage takes 0.31 us instead of 0.6 (its share of B is half, the ring
        // deeper): the parts' sums take 4 us through the cluster's shared memory for 128 rows and nearly none for one. K = 5120:
        // 1 row of 5120 columns takes 7.8 us by seven parts and 11.0 by pairs, 64 rows 8.9 and 11.4, 128 rows 11.0 and 11.7;
        // 128 rows of 15360 columns 18.4 by two parts and 14.8 by pairs, 300 rows of 5120 15.3 by parts and 12.8 by pairs.
        const long long stages = (p.K + KSTAGE - 1) / KSTAGE;
        if (split < 2 || stages * (split - 2) * 8 <= (long long)(std::min(p.M, BM) - 32) * split)
            return false;
        at[0].val.clusterDim.x = unsigned(split);
        ctas = tiles * split;
    }
    c.gridDim = dim3(unsigned(ctas));
    H3_CUDA(cudaLaunchKernelEx(&c, gemm_fp4_kernel<EPI, F, W>, in, p, om));
    return true;
}

template <Epi EPI, Fp4 F>
void run(const void* A, const void* a_scales, const void* B, const void* b_scales, const GemmParams& p, cudaStream_t s)
{
    const long long tiles_n = (p.N + BN - 1) / BN, tiles = (p.M + BM - 1) / BM * tiles_n;
    const int sms = num_sms();
    if constexpr (EPI != Epi::qkv) // its norm runs along whole rows of a tile
        if (tiles * 2 <= sms && p.K > KSTAGE && launch<EPI, F, Form::split>(A, a_scales, B, b_scales, p, int(tiles), sms, s))
            return;
    if (p.M > BM || tiles * 2 <= sms) {
        const long long pairs = (p.M + 2 * BM - 1) / (2 * BM) * tiles_n;
        launch<EPI, F, Form::pair>(A, a_scales, B, b_scales, p, int(pairs), int(std::min<long long>(pairs, sms / 2)) * 2, s);
    } else {
        launch<EPI, F, Form::tiles>(A, a_scales, B, b_scales, p, int(tiles), int(std::min<long long>(tiles, sms)), s);
    }
}

} // namespace

void gemm_fp4(const void* A, const void* a_scales, const void* B, const void* b_scales, Fp4 f, const GemmParams& p, Epi epi,
              cudaStream_t s)
{
    if (p.M <= 0)
        return;
    const bool nv = f == Fp4::nv;
    switch (epi) {
    case Epi::bf16: return (nv ? run<Epi::bf16, Fp4::nv> : run<Epi::bf16, Fp4::mx>)(A, a_scales, B, b_scales, p, s);
    case Epi::f32: return (nv ? run<Epi::f32, Fp4::nv> : run<Epi::f32, Fp4::mx>)(A, a_scales, B, b_scales, p, s);
    case Epi::qkv: return (nv ? run<Epi::qkv, Fp4::nv> : run<Epi::qkv, Fp4::mx>)(A, a_scales, B, b_scales, p, s);
    case Epi::gate_resid: return (nv ? run<Epi::gate_resid, Fp4::nv> : run<Epi::gate_resid, Fp4::mx>)(A, a_scales, B, b_scales, p, s);
    case Epi::swiglu: return (nv ? run<Epi::swiglu, Fp4::nv> : run<Epi::swiglu, Fp4::mx>)(A, a_scales, B, b_scales, p, s);
    default: throw std::runtime_error("gemm_fp4: unsupported epilogue");
    }
}

} // namespace h3
