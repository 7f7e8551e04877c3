// The projection GEMM on microscaled 4-bit rows (layouts in fp4.cuh): tcgen05.mma kind::mxf4 / kind::mxf4nvf4 with the
// block scales in TMEM, fp32 accumulation, the row scales and the step's epilogues on the way out.
//
// One persistent kernel, one CTA per SM, the roles of the bf16 GEMM: warp 0 loads (TMA tiles of 128 bytes = 256 values of
// K, 128-byte swizzled; the scale tiles by plain bulk copies), warp 1 issues, warps 2..5 are the epilogue. Per stage the
// issuing thread copies the stage's scale tiles from shared memory into TMEM (tcgen05.cp, in order before the MMAs that
// read them) and runs four M = 128, N = 256, K = 64 MMAs.
//
// TMEM: two accumulators of 256 columns and the scales do not fit 512 columns side by side, and N = 256 is what keeps the
// shared-memory reads of an MMA (12 KB) under its time, so the accumulators overlap in 96 columns:
//   [0, 256) accumulator 0, [160, 416) accumulator 1, [416, 512) two buffers of one stage's scales (48 columns each)
// An epilogue reads the shared columns first (into registers) and hands them on; the next tile's MMAs wait for that,
// not for the whole epilogue. A scale buffer is written again only after the MMAs that read it are known to be complete
// (the stage's `empty` barrier), two stages later: the stage between keeps the tensor core busy meanwhile.
#include "common.hpp"
#include "fp4.cuh"
#include "gemm_epi.cuh"
#include "ptx.cuh"

#include <algorithm>
#include <type_traits>

namespace h3 {

namespace {

constexpr int BM = 128, BN = 256;
constexpr int KSTAGE = 256;          // values of K per stage: 128 bytes of codes a row
constexpr int A_BYTES = BM * 128, B_BYTES = BN * 128;
constexpr int NUM_THREADS = 192;
constexpr int ACC1 = 160, OVERLAP = 96; // accumulator 1's first column, the columns that it shares with accumulator 0
constexpr int SCALE_COL = 416, SCALE_BUF = 48;

constexpr bool staged(Epi e) { return e == Epi::qkv || e == Epi::swiglu; } // output tiles through shared memory and TMA stores

template <Epi EPI, Fp4 F>
struct Fp4Smem {
    // scale tiles of a stage: 4 (nv) or 2 (mx) along K for A's 128 rows and twice as many for B's 256
    static constexpr int KT = KSTAGE / (4 * fp4_block(F));
    static constexpr int SF_BYTES = 3 * KT * 512;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + SF_BYTES;
    static constexpr int STAGING = staged(EPI) ? BM * 256 : 0;
    static constexpr int STAGES = staged(EPI) ? 3 : 4;
    static constexpr int TOTAL = STAGES * STAGE_BYTES + STAGING + 1024 + 256;
    static_assert(STAGE_BYTES % 1024 == 0 && TOTAL <= 227 * 1024);
};

struct NoMaps {};
template <Epi EPI>
using MapsOf = std::conditional_t<staged(EPI), OutMaps, NoMaps>;

// D[tmem] (+)= A[smem] B[smem]^T on e2m1 codes, the block scales in TMEM at sfa and sfb.
template <Fp4 F>
__device__ __forceinline__ void mma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate)
{
    if constexpr (F == Fp4::nv)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
                     "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
                     "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
                     : "memory");
}

// Instruction descriptor of the two kinds: e2m1 A and B, both K-major; the scales' type (1: powers of two, 0: e4m3) and
// which pair of the scale bytes of a TMEM word the MMA reads (mx: a word holds two MMAs' scales).
template <Fp4 F>
__device__ __forceinline__ constexpr uint32_t idesc_fp4(uint32_t pair)
{
    return (pair << 4) | (1u << 7) | (1u << 10) | (uint32_t(BN >> 3) << 17) | (uint32_t(F == Fp4::mx) << 23) | (uint32_t(BM >> 7) << 27) |
           (pair << 29);
}

// One scale tile (32 rows of 16 bytes in shared memory) into four TMEM columns of 32 lanes, repeated for the four
// 32-lane quarters.
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint32_t smem_addr)
{
    // 8-row groups of 128 bytes, no swizzle
    const uint64_t d = uint64_t((smem_addr >> 4) & 0x3FFF) | (uint64_t(128 >> 4) << 32) | (uint64_t(1) << 46);
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
}

// `CHUNKS` 32-column chunks of this thread's accumulator row, from column `col`, as they are.
template <int CHUNKS>
__device__ __forceinline__ void load_chunks(uint32_t taddr, int col, float* v)
{
    uint32_t r[CHUNKS][32];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
        tmem_ld32(taddr + col + c * 32, r[c]);
    tmem_wait_ld();
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int i = 0; i < 32; ++i)
            v[c * 32 + i] = __uint_as_float(r[c][i]);
}

// 32 columns from `col` times the row scales, plus the bias. Columns past N (whole groups of 8) are left alone.
__device__ __forceinline__ void finish_chunk(const GemmParams& p, float* v, int col, float a_scale)
{
    if (p.b_scale) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + 4 * i < p.N) {
                const float4 b = __ldg(reinterpret_cast<const float4*>(p.b_scale + col) + i);
                v[4 * i] *= a_scale * b.x, v[4 * i + 1] *= a_scale * b.y, v[4 * i + 2] *= a_scale * b.z, v[4 * i + 3] *= a_scale * b.w;
            }
    } else if (p.a_scale) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
            v[i] *= a_scale;
    }
    if (p.bias) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + 4 * i < p.N) {
                const float4 b = __ldg(reinterpret_cast<const float4*>(p.bias + col) + i);
                v[4 * i] += b.x, v[4 * i + 1] += b.y, v[4 * i + 2] += b.z, v[4 * i + 3] += b.w;
            }
    }
}

// The output of 32 finished columns of row gm (bf16, f32 and gated residual epilogues).
template <Epi EPI>
__device__ __forceinline__ void store_chunk(const GemmParams& p, const float* v, int gm, int col)
{
    if constexpr (EPI == Epi::bf16) {
        uint4* d = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + size_t(gm) * p.ldo + col);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (col + 8 * i < p.N)
                d[i] = make_uint4(pack_bf16x2(v[8 * i], v[8 * i + 1]), pack_bf16x2(v[8 * i + 2], v[8 * i + 3]),
                                  pack_bf16x2(v[8 * i + 4], v[8 * i + 5]), pack_bf16x2(v[8 * i + 6], v[8 * i + 7]));
    } else if constexpr (EPI == Epi::f32) {
        float4* d = reinterpret_cast<float4*>(static_cast<float*>(p.out) + size_t(gm) * p.ldo + col);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + 4 * i < p.N)
                d[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else {
        static_assert(EPI == Epi::gate_resid);
        const float4* g4 = reinterpret_cast<const float4*>(p.mod + (size_t(p.mod_idx[gm]) * 6 + p.gate_slot) * p.dim + col);
        float4* x4 = reinterpret_cast<float4*>(p.x + size_t(gm) * p.ldx + col);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + 4 * i < p.N) {
                const float4 g = __ldg(g4 + i);
                float4 x = x4[i];
                x.x += g.x * v[4 * i], x.y += g.y * v[4 * i + 1], x.z += g.z * v[4 * i + 2], x.w += g.w * v[4 * i + 3];
                x4[i] = x;
            }
    }
}

// Sixteen-byte piece `c` (8 columns) of a row's 128 staged bf16 columns (two 128-byte-swizzled halves).
__device__ __forceinline__ void stage_piece(uint8_t* stage, int row, int c, const float* v)
{
    *reinterpret_cast<uint4*>(stage + (c >> 3) * (BM * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4)) =
        make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

// The epilogue of one tile whose accumulator is number ACC. The columns that the other accumulator shares (the last 96 of
// accumulator 0, the first 96 of accumulator 1) are read first; `release` then lets the next tile's MMAs start.
template <Epi EPI, int ACC, class Release>
__device__ __forceinline__ void epilogue_fp4(const GemmParams& p, uint32_t tmem, int m0, int n0, uint8_t* stage, const MapsOf<EPI>& om,
                                             Release&& release)
{
    constexpr int FIRST = ACC == 0 ? ACC1 : 0; // first shared column of this accumulator
    const int quarter = warp_id() & 3;
    const int row = quarter * 32 + lane_id();
    const int gm = m0 + row;
    const bool valid = gm < p.M;
    const uint32_t taddr = tmem + (ACC == 0 ? 0 : ACC1) + (uint32_t(quarter * 32) << 16);
    const float a_scale = p.a_scale && valid ? __ldg(p.a_scale + gm) : 1.0f;

    if constexpr (EPI == Epi::qkv) {
        const int sec = n0 / p.inner;
        const int grow = valid ? gm : p.M - 1; // rows past M read a valid row's rotary entry
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
            const int hh = ACC == 0 ? 1 - i : i; // the head that lies in the shared columns first
            float v[128];
            load_chunks<4>(taddr, hh * 128, v);
            if (i == 0)
                release();
            const int col = n0 + hh * 128;
#pragma unroll
            for (int c = 0; c < 4; ++c)
                finish_chunk(p, v + 32 * c, col + 32 * c, a_scale);
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
                const float2* cs = reinterpret_cast<const float2*>(p.rope) + size_t(grow) * 48;
#pragma unroll
                for (int j = 0; j < 48; ++j) {
                    const float2 t = __ldg(cs + j);
                    const float a = v[j], b = v[j + 48];
                    v[j] = a * t.x - b * t.y;
                    v[j + 48] = b * t.x + a * t.y;
                }
            }
            const int head = (col % p.inner) / 128;
            const int rank = head / p.heads_per_rank, hl = head % p.heads_per_rank;
            if (threadIdx.x == 64)
                bulk_wait_read0(); // the staged tile before has been read
            epi_bar();
#pragma unroll
            for (int c = 0; c < 16; ++c)
                stage_piece(stage, row, c, v + 8 * c);
            fence_proxy_async_smem();
            epi_bar();
            if (threadIdx.x == 64) {
                const int slot = sec * p.heads_per_rank + hl;
                tma_store_3d(&om.m[rank], stage, 0, slot, m0);
                tma_store_3d(&om.m[rank], stage + BM * 128, 64, slot, m0);
                bulk_commit();
            }
        }
    } else if constexpr (EPI == Epi::swiglu) {
        // pair c: gate chunk c and value chunk c + 4; the shared columns hold the values of pairs 1..3 (accumulator 0) or the
        // gates of pairs 0..2 (accumulator 1)
        float held[OVERLAP];
        load_chunks<3>(taddr, FIRST, held);
        release();
        if (threadIdx.x == 64)
            bulk_wait_read0();
        epi_bar();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = ACC == 0 ? (i + 1) & 3 : i;
            float g[32], u[32];
            if (i < 3) {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    (ACC == 0 ? u : g)[j] = held[32 * i + j];
                load_chunks<1>(taddr, ACC == 0 ? c * 32 : 128 + c * 32, ACC == 0 ? g : u);
            } else {
                load_chunks<1>(taddr, c * 32, g);
                load_chunks<1>(taddr, 128 + c * 32, u);
            }
            finish_chunk(p, g, n0 + c * 32, a_scale);
            finish_chunk(p, u, n0 + 128 + c * 32, a_scale);
#pragma unroll
            for (int j = 0; j < 32; ++j)
                g[j] = silu(g[j]) * u[j];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                stage_piece(stage, row, c * 4 + j, g + 8 * j);
        }
        fence_proxy_async_smem();
        epi_bar();
        if (threadIdx.x == 64) {
            tma_store_2d(&om.m[0], stage, n0 / 2, m0);
            tma_store_2d(&om.m[0], stage + BM * 128, n0 / 2 + 64, m0);
            bulk_commit();
        }
    } else {
        float held[OVERLAP];
        load_chunks<3>(taddr, FIRST, held);
        release();
#pragma unroll
        for (int c = 0; c < 3; ++c) {
            const int col = n0 + FIRST + c * 32;
            if (valid && col < p.N) {
                finish_chunk(p, held + 32 * c, col, a_scale);
                store_chunk<EPI>(p, held + 32 * c, gm, col);
            }
        }
#pragma unroll 1
        for (int c = 0; c < 5; ++c) {
            const int at = (ACC == 0 ? 0 : OVERLAP) + c * 32, col = n0 + at;
            float v[32];
            load_chunks<1>(taddr, at, v);
            if (valid && col < p.N) {
                finish_chunk(p, v, col, a_scale);
                store_chunk<EPI>(p, v, gm, col);
            }
        }
    }
}

template <Epi EPI, Fp4 F>
__global__ void __launch_bounds__(NUM_THREADS, 1)
    gemm_fp4_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const uint8_t* a_scales,
                    const uint8_t* b_scales, const GemmParams p, const __grid_constant__ MapsOf<EPI> om)
{
    using SM = Fp4Smem<EPI, F>;
    constexpr int STAGES = SM::STAGES, KT = SM::KT;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t* smem = smem_raw + (((raw + 1023) & ~1023u) - raw);
    uint8_t* stage = smem + STAGES * SM::STAGE_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(stage + SM::STAGING);
    uint64_t* full = bars;              // [STAGES]
    uint64_t* empty = full + STAGES;    // [STAGES]
    uint64_t* tfull = empty + STAGES;   // [2] an accumulator is complete
    uint64_t* shared_free = tfull + 2;  // the shared columns of the tile before have been read
    uint64_t* drain = shared_free + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);

    const int warp = warp_id();
    const int tiles_m = (p.M + BM - 1) / BM, tiles_n = (p.N + BN - 1) / BN;
    const int num_tiles = tiles_m * tiles_n;
    const int num_kb = (p.K + KSTAGE - 1) / KSTAGE;
    const int scale_tiles = fp4_scale_tiles(p.K, F);

    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i)
            mbar_init(&tfull[i], 1);
        mbar_init(shared_free, 4);
        mbar_init(drain, 1);
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0 && elect_one_lane()) {
        // ---------------------------------------------------------------------------------------- producer
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
        uint32_t it = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
            int tm, tn;
            tile_coords(tile, tiles_m, tiles_n, tm, tn);
            const bool second = tn * BN + 128 < p.N; // B's second 128 rows have scale tiles
            for (int kb = 0; kb < num_kb; ++kb, ++it) {
                const int s = it % STAGES;
                if (!(ok = mbar_wait(&empty[s], ((it / STAGES) & 1) ^ 1)))
                    break;
                uint8_t* sa = smem + s * SM::STAGE_BYTES;
                uint8_t* sb = sa + A_BYTES;
                uint8_t* sf = sb + B_BYTES;
                const uint32_t sf_bytes = uint32_t(min(KT, scale_tiles - kb * KT)) * 512;
                mbar_arrive_expect_tx(&full[s], A_BYTES + B_BYTES + sf_bytes * (second ? 3 : 2));
                tma_load_2d(sa, &tmA, &full[s], kb * 128, tm * BM);
                tma_load_2d(sb, &tmB, &full[s], kb * 128, tn * BN);
                bulk_load(sf, a_scales + (size_t(tm) * scale_tiles + kb * KT) * 512, sf_bytes, &full[s]);
                bulk_load(sf + KT * 512, b_scales + (size_t(2 * tn) * scale_tiles + kb * KT) * 512, sf_bytes, &full[s]);
                if (second)
                    bulk_load(sf + 2 * KT * 512, b_scales + (size_t(2 * tn + 1) * scale_tiles + kb * KT) * 512, sf_bytes, &full[s]);
            }
        }
        // Wait for the loads still in flight to land before the CTA can exit.
        if (ok)
            for (uint32_t j = it >= STAGES ? it - STAGES : 0; j < it; ++j)
                mbar_wait(&empty[j % STAGES], (j / STAGES) & 1);
    } else if (warp == 1 && elect_one_lane()) {
        // ------------------------------------------------------------------------------------- MMA issuer
        uint32_t it = 0, t_local = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x, ++t_local) {
            // the tile before has left the columns that both accumulators use (and, as its epilogue came after that of the
            // tile before it, this accumulator is free)
            if (t_local > 0 && !(ok = mbar_wait(shared_free, (t_local - 1) & 1)))
                break;
            tc_fence_after();
            const uint32_t d = tmem + (t_local & 1) * ACC1;
            for (int kb = 0; kb < num_kb; ++kb, ++it) {
                const int s = it % STAGES;
                if (!(ok = mbar_wait(&full[s], (it / STAGES) & 1)))
                    break;
                // the MMAs of two stages ago, which read this scale buffer, are complete
                if (it >= 2 && !(ok = mbar_wait(&empty[(it - 2) % STAGES], ((it - 2) / STAGES) & 1)))
                    break;
                tc_fence_after();
                const uint32_t sa = smem_u32(smem + s * SM::STAGE_BYTES);
                const uint32_t sb = sa + A_BYTES, sf = sb + B_BYTES;
                const uint32_t tsf = tmem + SCALE_COL + (it & 1) * SCALE_BUF;
                const int steps = min(KSTAGE, p.K - kb * KSTAGE + 63) / 64; // MMAs of this stage (64 values each)
                const int kts = min(KT, scale_tiles - kb * KT);
                for (int k = 0; k < kts; ++k) {
                    copy_scales(tsf + k * 12, sf + k * 512);
                    copy_scales(tsf + k * 12 + 4, sf + (KT + k) * 512);
                    copy_scales(tsf + k * 12 + 8, sf + (2 * KT + k) * 512);
                }
#pragma unroll
                for (int k = 0; k < KSTAGE / 64; ++k) {
                    if (k >= steps)
                        break;
                    const uint64_t ad = sdesc_sw128(sa + k * 32, 16, 1024);
                    const uint64_t bd = sdesc_sw128(sb + k * 32, 16, 1024);
                    const uint32_t kt = F == Fp4::nv ? k : k / 2;
                    mma_fp4<F>(d, ad, bd, idesc_fp4<F>(F == Fp4::nv ? 0 : (k & 1) * 2), tsf + kt * 12, tsf + kt * 12 + 4, (kb | k) != 0);
                }
                mma_commit(&empty[s]);
            }
            if (ok)
                mma_commit(&tfull[t_local & 1]);
        }
        // Every MMA this thread issued has completed once `drain` flips.
        mma_commit(drain);
        mbar_wait(drain, 0);
    } else if (warp >= 2) {
        // ---------------------------------------------------------------------------------------- epilogue
        uint32_t t_local = 0;
        auto release = [&] {
            tc_fence_before();
            __syncwarp();
            if (elect_one_lane())
                mbar_arrive(shared_free);
        };
        for (int tile = blockIdx.x; tile < num_tiles; tile += gridDim.x, ++t_local) {
            const int acc = t_local & 1;
            if (!mbar_wait(&tfull[acc], (t_local >> 1) & 1))
                break;
            tc_fence_after();
            int tm, tn;
            tile_coords(tile, tiles_m, tiles_n, tm, tn);
            if (acc == 0)
                epilogue_fp4<EPI, 0>(p, tmem, tm * BM, tn * BN, stage, om, release);
            else
                epilogue_fp4<EPI, 1>(p, tmem, tm * BM, tn * BN, stage, om, release);
        }
        if (staged(EPI) && threadIdx.x == 64)
            bulk_wait0(); // the staged tiles' TMA stores are complete
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <Epi EPI, Fp4 F>
void launch(const void* A, const void* a_scales, const void* B, const void* b_scales, const GemmParams& p, cudaStream_t s)
{
    using SM = Fp4Smem<EPI, F>;
    const uint64_t bytes = uint64_t(p.K) / 2;
    const uint64_t adims[2] = {bytes, uint64_t(p.M)}, bdims[2] = {bytes, uint64_t(p.N)}, pitch[1] = {bytes};
    const uint32_t abox[2] = {128, BM}, bbox[2] = {128, BN};
    const CUtensorMap ta = make_tmap(CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, A, adims, pitch, abox);
    const CUtensorMap tb = make_tmap(CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, B, bdims, pitch, bbox);
    MapsOf<EPI> om{};
    if constexpr (staged(EPI))
        om = out_maps<EPI>(p, p.M);
    static std::atomic<uint64_t> opt_in;
    smem_opt_in(gemm_fp4_kernel<EPI, F>, SM::TOTAL, opt_in);
    const long long tiles = (long long)((p.M + BM - 1) / BM) * ((p.N + BN - 1) / BN);
    const int grid = int(std::min<long long>(tiles, num_sms()));
    gemm_fp4_kernel<EPI, F><<<grid, NUM_THREADS, SM::TOTAL, s>>>(ta, tb, static_cast<const uint8_t*>(a_scales),
                                                                 static_cast<const uint8_t*>(b_scales), p, om);
    H3_CUDA(cudaGetLastError());
}

} // namespace

void gemm_fp4(const void* A, const void* a_scales, const void* B, const void* b_scales, Fp4 f, const GemmParams& p, Epi epi,
              cudaStream_t s)
{
    if (p.M <= 0)
        return;
    const bool nv = f == Fp4::nv;
    switch (epi) {
    case Epi::bf16: return (nv ? launch<Epi::bf16, Fp4::nv> : launch<Epi::bf16, Fp4::mx>)(A, a_scales, B, b_scales, p, s);
    case Epi::f32: return (nv ? launch<Epi::f32, Fp4::nv> : launch<Epi::f32, Fp4::mx>)(A, a_scales, B, b_scales, p, s);
    case Epi::qkv: return (nv ? launch<Epi::qkv, Fp4::nv> : launch<Epi::qkv, Fp4::mx>)(A, a_scales, B, b_scales, p, s);
    case Epi::gate_resid: return (nv ? launch<Epi::gate_resid, Fp4::nv> : launch<Epi::gate_resid, Fp4::mx>)(A, a_scales, B, b_scales, p, s);
    case Epi::swiglu: return (nv ? launch<Epi::swiglu, Fp4::nv> : launch<Epi::swiglu, Fp4::mx>)(A, a_scales, B, b_scales, p, s);
    default: throw std::runtime_error("gemm_fp4: unsupported epilogue");
    }
}

} // namespace h3
