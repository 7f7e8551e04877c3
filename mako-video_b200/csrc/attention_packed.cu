// Flash attention over packed documents on sm_100a: o_i = sum_j p_ij v_j / sum_j p_ij with p_ij = 2^(s_ij - m_i), the sum
// over the keys of row i's document and the shared prefix, one pass over the keys with a running maximum m_i.
//
// The pipeline is the dense kernel's (attention.cu): per CTA two 128-row query tiles of one kv head share each K/V tile; S and
// O in TMEM, P written back over S and read from there by the PV MMA; O rescaled only when a row's maximum grows by more
// than 2^8. What differs:
//   - A CTA is a run of query rows of one document. Launches have a slot for every run that the documents could need
//     (a document of rows [a, b) owns the slots from a / TR + d on, TR rows a run), so the host needs no lengths; a slot
//     without rows ends at once.
//   - The `group` query heads of a kv head are stacked into the tile's rows (row r of the tile: query row r / group, head
//     r % group, by the TMA box alone), so shared keys are loaded once for all of them, and one query row of a large
//     group fills a tile.
//   - Keys come as the prefix's 128-row blocks, then the document's own (one run where they adjoin). Rows of a block past
//     its end belong to someone else and may hold anything: their scores are replaced, and their V rows are zeroed in
//     shared memory (0 x NaN is a NaN) by tile 0's softmax warps before they hand over P.
//   - With few runs the keys are split over the CTAs of a cluster, and the parts joined through shared memory of the
//     cluster: no scratch in HBM, no second launch, a fixed order of the sums.
#include "attention_packed.cuh"
#include "common.hpp"
#include "ptx.cuh"

#include <algorithm>
#include <cmath>
#include <cuda_fp16.h>

namespace h3 {

namespace {

constexpr int HALF = 16384;                // 128 rows x 64 dims of 2 bytes
constexpr float kRescaleThreshold = 8.0f;  // log2 units
constexpr int KST = 3, VST = 2;            // K is freed once both S MMAs read it, V after both PV MMAs
constexpr int NT = 64 + 256;

template <int HD>
struct PkSmem {
    static constexpr int TL = 128 * HD * 2; // a 128-row tile of one head
    static constexpr int OFF_K = 2 * TL;    // Q0, Q1 first
    static constexpr int OFF_V = OFF_K + KST * TL;
    static constexpr int OFF_BAR = OFF_V + VST * TL;
    static constexpr int TOTAL = OFF_BAR + 256 + 1024;
    // a split launch's parts: [256 rows][HD] fp32 over the K/V rings, (max, sum) of the rows over Q
    static_assert(256 * HD * 4 <= (KST + VST) * TL && 256 * 8 <= 2 * TL);
};

struct PkMaps {
    CUtensorMap q, k, v; // (dim, head, row): boxes 64 x group x rows per 64-row unit, 64 x 1 x 64
};

struct PkArgs {
    void* out;
    int64_t out_stride;
    const int32_t* q_start;
    const int32_t* k_start;
    int q_rows, k_rows, docs, prefix, group, unit_rows; // unit_rows: query rows in a 64-row unit, 64 / group
    float sl2;                                          // scale log2(e)
};

template <bool F16>
__host__ __device__ constexpr uint32_t idesc_16(int M, int N, bool b_mn)
{
    return (1u << 4) | (F16 ? 0u : (1u << 7) | (1u << 10)) | (uint32_t(b_mn) << 16) | (uint32_t(N >> 3) << 17) | (uint32_t(M >> 4) << 24);
}

template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    if constexpr (F16) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        return pack_bf16x2(lo, hi);
    }
}

__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// Reads shared memory of CTA `rank` of the cluster at this CTA's address `addr`.
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr, uint32_t rank)
{
    float4 v;
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\tld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n\t}"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr), "r"(rank)
                 : "memory");
    return v;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t addr, uint32_t rank)
{
    float2 v;
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %2, %3;\n\tld.shared::cluster.v2.f32 {%0, %1}, [a];\n\t}"
                 : "=f"(v.x), "=f"(v.y)
                 : "r"(addr), "r"(rank)
                 : "memory");
    return v;
}

// The document whose slots hold `slot`, or -1: the last d with q_start[d] / run + d <= slot. One warp, 32 candidates a step.
__device__ __forceinline__ int find_document(const PkArgs& p, int slot, int run)
{
    int lo = 0, n = p.docs;
    while (true) {
        const int step = (n + 31) / 32;
        const int d = lo + lane_id() * step;
        const bool before = lane_id() * step < n && min(max(__ldg(p.q_start + d), 0), p.q_rows) / run + d <= slot;
        const uint32_t yes = __ballot_sync(0xffffffffu, before);
        if (!yes)
            return -1; // rows before the first document
        const int k = 31 - __clz(yes);
        lo += k * step;
        n = min(step, n - k * step);
        if (step == 1)
            return lo;
    }
}

template <int HD, bool F16>
__global__ void __launch_bounds__(NT, 1) packed_attention_kernel(const __grid_constant__ PkMaps maps, const PkArgs p)
{
    using SM = PkSmem<HD>;
    constexpr int TL = SM::TL, OFF_K = SM::OFF_K, OFF_V = SM::OFF_V;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t* smem = smem_raw + (((raw + 1023) & ~1023u) - raw);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + SM::OFF_BAR);
    uint64_t* q_full = bars + 0;
    uint64_t* k_full = bars + 1;       // [KST]
    uint64_t* k_empty = k_full + KST;  // [KST]
    uint64_t* v_full = k_empty + KST;  // [VST]
    uint64_t* v_empty = v_full + VST;  // [VST]
    uint64_t* s_full = v_empty + VST;  // [2] per tile
    uint64_t* p_full = s_full + 2;     // [2] per tile
    uint64_t* pv_done = p_full + 2;    // [2] per tile
    uint64_t* drain = pv_done + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);

    const int warp = warp_id();
    uint32_t split, part; // CTAs of this run's cluster, this one's number
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(split));
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(part));
    const int slot = blockIdx.x / split, kv_head = blockIdx.y;
    const int run = 4 * p.unit_rows;

    if (blockIdx.x == 0 && blockIdx.y == 0) // the starts ascend within the tensors; a document with others is left out
        for (int d = threadIdx.x; d <= p.docs; d += NT) {
            const int a = p.q_start[d], b = p.k_start[d];
            if (a < 0 || a > p.q_rows || b < 0 || b > p.k_rows || (d > 0 && (a < p.q_start[d - 1] || b < p.k_start[d - 1])))
                record_error(kErrBadShape);
        }

    // This CTA's query rows [row0, q1) and the keys [0, a_end) and [b0, b_end) of their document.
    const int doc = find_document(p, slot, run);
    if (doc < 0)
        return;
    const int q0 = __ldg(p.q_start + doc), q1 = __ldg(p.q_start + doc + 1);
    const int row0 = q0 + (slot - (q0 / run + doc)) * run;
    int b0 = __ldg(p.k_start + doc), b_end = __ldg(p.k_start + doc + 1);
    if (q0 < 0 || row0 < q0 || row0 >= q1 || q1 > p.q_rows || b0 < 0 || b_end < b0 || b_end > p.k_rows)
        return;
    int a_end = p.prefix;
    b0 = max(b0, p.prefix);
    b_end = max(b_end, b0);
    if (b0 == p.prefix)
        a_end = b_end, b0 = b_end; // the document's keys adjoin the prefix: one run
    const int a_blocks = (a_end + 127) / 128;
    const int blocks = a_blocks + (b_end - b0 + 127) / 128;
    const int per = (blocks + int(split) - 1) / int(split);
    const int first = min(int(part) * per, blocks);
    const int nkv = min(per, blocks - first); // this CTA's blocks [first, first + nkv)
    // first row and rows of this CTA's block j
    auto block_row = [&](int j) { return first + j < a_blocks ? 128 * (first + j) : b0 + 128 * (first + j - a_blocks); };
    auto block_keys = [&](int j) { return min(128, (first + j < a_blocks ? a_end : b_end) - block_row(j)); };
    const bool two = row0 + 2 * p.unit_rows < q1; // the second tile has rows

    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        for (int i = 0; i < KST; ++i) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], 1);
        }
        for (int i = 0; i < VST; ++i) {
            mbar_init(&v_full[i], 1);
            mbar_init(&v_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&pv_done[i], 1);
        }
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
        // ------------------------------------------------------------------------------------------ TMA
        const int units = two ? 4 : 2;
        bool ok = true;
        if (nkv > 0) {
            mbar_arrive_expect_tx(q_full, uint32_t(units * p.unit_rows * p.group * HD * 2));
            for (int u = 0; u < units; ++u)
                for (int hh = 0; hh < HD / 64; ++hh)
                    tma_load_3d(smem + (u >> 1) * TL + hh * HALF + (u & 1) * 8192, &maps.q, q_full, hh * 64, kv_head * p.group,
                                row0 + u * p.unit_rows);
        }
        auto load = [&](uint8_t* tile, const CUtensorMap* map, uint64_t* bar, int j) {
            mbar_arrive_expect_tx(bar, TL);
            const int row = block_row(j);
#pragma unroll
            for (int hh = 0; hh < HD / 64; ++hh) {
                tma_load_3d(tile + hh * HALF, map, bar, hh * 64, kv_head, row);
                tma_load_3d(tile + hh * HALF + 8192, map, bar, hh * 64, kv_head, row + 64);
            }
        };
        // K runs ahead of V by up to the depth of its ring
        int jk = 0, jv = 0;
        while (jv < nkv) {
            if (jk < nkv && jk < jv + KST) {
                const int s = jk % KST;
                if (!(ok = mbar_wait(&k_empty[s], ((jk / KST) & 1) ^ 1)))
                    break;
                load(smem + OFF_K + s * TL, &maps.k, &k_full[s], jk);
                ++jk;
            } else {
                const int s = jv % VST;
                if (!(ok = mbar_wait(&v_empty[s], ((jv / VST) & 1) ^ 1)))
                    break;
                load(smem + OFF_V + s * TL, &maps.v, &v_full[s], jv);
                ++jv;
            }
        }
        // Loads that no one waited for (a pipeline that gave up) land before the CTA can exit.
        if (nkv > 0)
            mbar_wait(q_full, 0);
        for (int j = max(0, jk - KST); j < jk; ++j)
            mbar_wait(&k_full[j % KST], (j / KST) & 1);
        for (int j = max(0, jv - VST); j < jv; ++j)
            mbar_wait(&v_full[j % VST], (j / VST) & 1);
    } else if (warp == 1 && elect_one_lane()) {
        // ------------------------------------------------------------------------------------------ MMA
        const uint32_t id_s = idesc_16<F16>(128, 128, false);
        const uint32_t id_pv = idesc_16<F16>(128, HD, true);
        auto issue_s = [&](int t, int j) {
            const int ks = j % KST;
            const uint32_t sq = smem_u32(smem + t * TL);
            const uint32_t sk = smem_u32(smem + OFF_K + ks * TL);
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk) {
                const uint32_t off = (kk >> 2) * HALF + (kk & 3) * 32;
                mma_bf16_ss(tmem + t * 128, sdesc_sw128(sq + off, 16, 1024), sdesc_sw128(sk + off, 16, 1024), id_s, kk > 0);
            }
            mma_commit(&s_full[t]);
            if (t == 1 || !two)
                mma_commit(&k_empty[ks]); // every tile's S MMAs have read K_j
        };
        auto issue_pv = [&](int t, int j) {
            const int vs = j % VST;
            const uint32_t sv = smem_u32(smem + OFF_V + vs * TL);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)
                mma_bf16_ts(tmem + 256 + t * HD, tmem + t * 128 + kk * 8, sdesc_sw128(sv + kk * 2048, HALF, 1024), id_pv, (j | kk) != 0);
            mma_commit(&pv_done[t]);
            if (t == 1 || !two)
                mma_commit(&v_empty[vs]); // every tile's PV MMAs have read V_j
        };
        bool ok = nkv > 0 && mbar_wait(q_full, 0) && mbar_wait(&k_full[0], 0);
        if (ok) {
            tc_fence_after();
            issue_s(0, 0);
            if (two)
                issue_s(1, 0);
        }
        for (int j = 0; j < nkv && ok; ++j) {
            if (!(ok = mbar_wait(&v_full[j % VST], (j / VST) & 1) && mbar_wait(&p_full[0], j & 1)))
                break;
            tc_fence_after();
            issue_pv(0, j);
            const bool more = j + 1 < nkv;
            if (more) {
                if (!(ok = mbar_wait(&k_full[(j + 1) % KST], ((j + 1) / KST) & 1)))
                    break;
                tc_fence_after();
                issue_s(0, j + 1);
            }
            if (two) {
                if (!(ok = mbar_wait(&p_full[1], j & 1)))
                    break;
                tc_fence_after();
                issue_pv(1, j);
                if (more)
                    issue_s(1, j + 1);
            }
        }
        mma_commit(drain);
        mbar_wait(drain, 0);
    } else if (warp >= 2 && (two || warp < 6)) {
        // -------------------------------------------------------------------------------------- softmax
        const int t = (warp - 2) / 4;
        const int quarter = warp & 3;
        const int row = quarter * 32 + lane_id();
        const uint32_t lane_base = uint32_t(quarter * 32) << 16;
        const uint32_t tS = tmem + lane_base + t * 128;
        const uint32_t tO = tmem + lane_base + 256 + t * HD;
        // this thread's query row and head
        const int in_unit = row & 63;
        const int out_row = row0 + (2 * t + (row >> 6)) * p.unit_rows + in_unit / p.group;
        const bool valid = in_unit < p.unit_rows * p.group && out_row < q1;
        const bool idle = !__any_sync(0xffffffffu, valid); // rows that nobody asked for: their P may be anything
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int j = 0; j < nkv; ++j) {
            if (!(ok = mbar_wait(&s_full[t], j & 1)))
                break;
            tc_fence_after();
            const int keys = block_keys(j);
            if (t == 0 && keys < 128) {
                // V rows past the block's keys
                if (!(ok = mbar_wait(&v_full[j % VST], (j / VST) & 1)))
                    break;
                uint8_t* sv = smem + OFF_V + (j % VST) * TL;
                for (int i = keys * 8 + row; i < 128 * 8; i += 128)
#pragma unroll
                    for (int hh = 0; hh < HD / 64; ++hh)
                        *reinterpret_cast<uint4*>(sv + hh * HALF + i * 16) = make_uint4(0, 0, 0, 0);
                fence_proxy_async_smem();
            }
            if (!idle) {
                float s[128];
                {
                    uint32_t r[4][32];
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        tmem_ld32(tS + c * 32, r[c]);
                    tmem_wait_ld();
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            s[c * 32 + i] = __uint_as_float(r[c][i]);
                }
                if (keys < 128) {
#pragma unroll
                    for (int c = 0; c < 128; ++c)
                        if (c >= keys)
                            s[c] = -INFINITY;
                }
                float mp[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    mp[i] = fmaxf(s[2 * i], s[2 * i + 1]);
#pragma unroll
                for (int c = 16; c < 128; c += 16)
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        mp[i] = max3f(mp[i], s[c + 2 * i], s[c + 2 * i + 1]);
                const float mx = max3f(max3f(mp[0], mp[1], mp[2]), max3f(mp[3], mp[4], mp[5]), fmaxf(mp[6], mp[7]));
                const float m_cand = mx * p.sl2;
                const bool need = m_cand > m + kRescaleThreshold;
                const float m_use = need ? m_cand : m;
                const float alpha = need ? ex2_approx(m - m_use) : 1.f;
                const float msub = m_use == -INFINITY ? 0.f : m_use;
                const float2 scale2 = make_float2(p.sl2, p.sl2), neg2 = make_float2(-msub, -msub);
                float2 sp[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                uint32_t pk[64]; // P rounded to the values' type for the tensor core; the row sum takes the unrounded ones
#pragma unroll
                for (int c = 0; c < 64; ++c) {
                    const float2 x = fma2(make_float2(s[2 * c], s[2 * c + 1]), scale2, neg2);
                    const float2 e = make_float2(ex2_approx(x.x), ex2_approx(x.y));
                    sp[c & 3] = add2(sp[c & 3], e);
                    pk[c] = pack2<F16>(e.x, e.y);
                }
                const float2 s01 = add2(add2(sp[0], sp[1]), add2(sp[2], sp[3]));
                if (j > 0 && __any_sync(0xffffffffu, need)) {
                    // O_t holds PV_t(0..j-1), complete (S_t(j) was issued after PV_t(j-1))
#pragma unroll 1
                    for (int c = 0; c < HD / 32; ++c) {
                        uint32_t o[32];
                        tmem_ld32(tO + c * 32, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                        tmem_st32(tO + c * 32, o);
                    }
                }
                l = l * alpha + (s01.x + s01.y);
                m = m_use;
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    tmem_st32(tS + c * 32, *reinterpret_cast<uint32_t(*)[32]>(pk + c * 32));
                tmem_wait_st();
            }
            tc_fence_before();
            __syncwarp();
            if (elect_one_lane())
                mbar_arrive(&p_full[t]);
        }
        const bool done = ok && (nkv == 0 || mbar_wait(&pv_done[t], (nkv - 1) & 1));
        tc_fence_after();
        if (split > 1) {
            // This part's unnormalised rows and their (max, sum), for the join below. A part that gave up counts for
            // nothing (the device error says so); one without keys too.
            const bool have = done && nkv > 0;
            float2* ml = reinterpret_cast<float2*>(smem) + t * 128 + row;
            float* o_row = reinterpret_cast<float*>(smem + OFF_K) + size_t(t * 128 + row) * HD;
            // Q and the rings are read by MMAs that are complete for this tile only: wait for the other one too
            const bool all = have && (!two || mbar_wait(&pv_done[t ^ 1], (nkv - 1) & 1));
            if (!idle) {
                *ml = all ? make_float2(m, l) : make_float2(-INFINITY, 0.f);
                if (all) {
#pragma unroll 1
                    for (int c = 0; c < HD / 32; ++c) {
                        uint32_t o[32];
                        tmem_ld32(tO + c * 32, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 8; ++i) // 16-byte pieces swizzled over the banks
                            *reinterpret_cast<float4*>(o_row + (((c * 8 + i) ^ (row & 7)) << 2)) =
                                make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]),
                                            __uint_as_float(o[4 * i + 3]));
                    }
                }
            }
        } else if (done && !idle) {
            const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l); // no key (or none above -infinity): 0; a NaN stays one
            uint16_t* dst = static_cast<uint16_t*>(p.out) + size_t(out_row) * p.out_stride + (kv_head * p.group + in_unit % p.group) * HD;
#pragma unroll 1
            for (int c = 0; c < HD / 32; ++c) {
                uint32_t o[32];
                if (nkv > 0) {
                    tmem_ld32(tO + c * 32, o);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        o[i] = 0;
                }
                if (valid) {
                    uint4* d4 = reinterpret_cast<uint4*>(dst + c * 32);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        d4[i] = make_uint4(pack2<F16>(__uint_as_float(o[8 * i]) * inv, __uint_as_float(o[8 * i + 1]) * inv),
                                           pack2<F16>(__uint_as_float(o[8 * i + 2]) * inv, __uint_as_float(o[8 * i + 3]) * inv),
                                           pack2<F16>(__uint_as_float(o[8 * i + 4]) * inv, __uint_as_float(o[8 * i + 5]) * inv),
                                           pack2<F16>(__uint_as_float(o[8 * i + 6]) * inv, __uint_as_float(o[8 * i + 7]) * inv));
                }
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
    if (split > 1) {
        // Join: a warp a row, the rows dealt out over the cluster's CTAs; parts weighted by 2^(m_part - max), in their order.
        cluster_sync();
        const int rows = two ? 256 : 128;
        for (int r = int(part) + warp * int(split); r < rows; r += int(split) * (NT / 32)) {
            const int in_unit = r & 63;
            const int out_row = row0 + (r >> 6) * p.unit_rows + in_unit / p.group;
            if (in_unit >= p.unit_rows * p.group || out_row >= q1)
                continue;
            const uint32_t ml = smem_u32(smem) + r * 8;
            float mx = -INFINITY;
            for (uint32_t z = 0; z < split; ++z)
                mx = fmaxf(mx, ld_cluster2(ml, z).x);
            const float sub = mx == -INFINITY ? 0.f : mx;
            float sum = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            const int piece = lane_id() < HD / 4 ? lane_id() : 0;
            const uint32_t o = smem_u32(smem + OFF_K) + r * HD * 4 + ((piece ^ (r & 7)) << 4);
            for (uint32_t z = 0; z < split; ++z) {
                const float2 a = ld_cluster2(ml, z);
                if (a.y == 0.f)
                    continue; // a part without keys has written no row
                const float w = ex2_approx(a.x - sub);
                const float4 v = ld_cluster4(o, z);
                sum += w * a.y;
                acc.x += w * v.x, acc.y += w * v.y, acc.z += w * v.z, acc.w += w * v.w;
            }
            const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
            if (lane_id() < HD / 4) {
                uint16_t* dst = static_cast<uint16_t*>(p.out) + size_t(out_row) * p.out_stride + (kv_head * p.group + in_unit % p.group) * HD;
                *reinterpret_cast<uint2*>(dst + piece * 4) = make_uint2(pack2<F16>(acc.x * inv, acc.y * inv), pack2<F16>(acc.z * inv, acc.w * inv));
            }
        }
        cluster_sync(); // no CTA leaves while another reads its shared memory
    }
}

CUtensorMap rows_map(const void* base, bool f16, int heads, int rows, int64_t stride, int head_dim, int box_heads, int box_rows)
{
    const uint64_t dims[3] = {uint64_t(head_dim), uint64_t(heads), uint64_t(rows)};
    const uint64_t str[2] = {uint64_t(head_dim) * 2, uint64_t(rows > 1 ? stride : int64_t(heads) * head_dim) * 2};
    const uint32_t box[3] = {64, uint32_t(box_heads), uint32_t(box_rows)};
    return make_tmap(f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, base, dims, str, box);
}

template <int HD, bool F16>
void launch(const PkMaps& maps, const PkArgs& a, int slots, int kv_heads, int split, cudaStream_t s)
{
    static std::atomic<uint64_t> opt_in;
    smem_opt_in(packed_attention_kernel<HD, F16>, PkSmem<HD>::TOTAL, opt_in);
    cudaLaunchConfig_t c{};
    c.gridDim = dim3(unsigned(slots) * split, kv_heads);
    c.blockDim = dim3(NT);
    c.dynamicSmemBytes = PkSmem<HD>::TOTAL;
    c.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = unsigned(split), at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    c.attrs = at;
    c.numAttrs = 1;
    H3_CUDA(cudaLaunchKernelEx(&c, packed_attention_kernel<HD, F16>, maps, a));
}

} // namespace

void attention_packed(const PackedAttnParams& p, cudaStream_t s)
{
    const int group = p.heads / p.kv_heads, unit_rows = 64 / group, run = 4 * unit_rows;
    PkMaps maps;
    maps.q = rows_map(p.q, p.f16, p.heads, p.q_rows, p.q_stride, p.head_dim, group, unit_rows);
    // without key rows there is nothing to describe, and no load is made
    maps.k = p.k_rows > 0 ? rows_map(p.k, p.f16, p.kv_heads, p.k_rows, p.k_stride, p.head_dim, 1, 64) : maps.q;
    maps.v = p.k_rows > 0 ? rows_map(p.v, p.f16, p.kv_heads, p.k_rows, p.v_stride, p.head_dim, 1, 64) : maps.q;
    PkArgs a{};
    a.out = p.out, a.out_stride = p.out_stride, a.q_start = p.q_start, a.k_start = p.k_start, a.q_rows = p.q_rows, a.k_rows = p.k_rows;
    a.docs = p.docs, a.prefix = p.prefix, a.group = group, a.unit_rows = unit_rows;
    a.sl2 = float(double(p.scale) * 1.4426950408889634);
    // Every run of every document has a slot: a / run + d is a document's first, and the last is at most this.
    const int slots = p.q_rows / run + p.docs;
    // Split the keys while the CTAs would still fit the SMs at once and each keeps four blocks of keys.
    const long long runs = std::max<long long>(p.docs, (p.q_rows + run - 1) / run);
    const long long blocks = (p.prefix + (p.k_rows - p.prefix) / p.docs + 127) / 128;
    int split = 1;
    while (split < 8 && runs * p.kv_heads * split * 2 <= num_sms() && blocks >= split * 8)
        split *= 2;
    if (p.head_dim == 128)
        (p.f16 ? launch<128, true> : launch<128, false>)(maps, a, slots, p.kv_heads, split, s);
    else
        (p.f16 ? launch<64, true> : launch<64, false>)(maps, a, slots, p.kv_heads, split, s);
}

} // namespace h3
