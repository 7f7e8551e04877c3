// Flash attention over packed documents on sm_100a: o_i = sum_j p_ij v_j / sum_j p_ij with p_ij = 2^(s_ij - m_i), the sum
// over the keys of row i's document and the shared prefix, one pass over the keys with a running maximum m_i.
//
// The pipeline is the dense kernel's (attention.cu): per CTA two 128-row query tiles of one kv head share each K/V tile; S and
// O in TMEM, P written back over S and read from there by the PV MMA; O rescaled only when a row's maximum grows by more
// than 2^8. What differs:
//   - A CTA is a run of query rows of one document. Launches have a slot for every run that the documents could need
//     (rows / TR + documents, TR rows a run), so the host needs no lengths; a slot without rows ends at once. Up to 32
//     documents get their slots in the order of their keys, longest first, which leaves short runs for the end of a
//     launch; of more, document d owns the slots from q_start[d] / TR + d on.
//   - The `group` query heads of a kv head are stacked into the tile's rows (row r of the tile: query row r / group, head
//     r % group, by the TMA box alone), so shared keys are loaded once for all of them, and one query row of a large
//     group fills a tile.
//   - Keys come as the prefix's 128-row blocks, then the document's own (one run where they adjoin). Rows of a block past
//     its end belong to someone else and may hold anything: their scores are replaced, and their V rows are zeroed in
//     shared memory (0 x NaN is a NaN) by tile 0's softmax warps before they hand over P.
//   - A run that fills one tile only has its even key blocks in one tile's place and its odd ones in the other's, so that
//     the two still overlap (a row's keys then come in two parts).
//   - With few runs the keys are split over the CTAs of a cluster. Parts are joined through the cluster's shared memory: no
//     scratch in HBM, no second launch, a fixed order of the sums.
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
// K and V slots. K is freed once its S MMAs have read it, V after its PV MMAs. With one query tile its room for a second
// one is a third V slot.
constexpr int KST = 3, VST = 2;
constexpr int NT = 64 + 256;
// 128-key blocks of a CTA's before more of its cluster join in, and of theirs at least: a block of two query tiles takes 1.9 us, writing,
// joining and storing the parts of 256 rows about 8 (256 rows of 10 heads of 128 on 1000 keys in 22.2 us by one CTA, 21.4 by two; on
// 3000 keys in 50.7 by one, 29.3 by three, 24.3 by six).
constexpr int LEAST = 4;
constexpr int MAX_SPLIT = 8; // CTAs of a cluster

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
    int32_t* status;
    int q_rows, k_rows, kv_heads, docs, prefix, group, unit_rows; // unit_rows: query rows in a 64-row unit, 64 / group
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

// -infinity in this warp's lanes of the TMEM columns [from, 128) after `taddr`. (Masking the scores in registers instead
// costs every step their spills.)
__device__ __forceinline__ void hide_columns(uint32_t taddr, int from)
{
    const uint32_t inf = 0xff800000u;
    int c = from;
    for (; c & 7; ++c)
        asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(taddr + c), "r"(inf));
    for (; c < 128; c += 8)
        asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %1, %1, %1, %1, %1, %1, %1};" ::"r"(taddr + c), "r"(inf));
    tmem_wait_st();
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

struct Document {
    int index, tile; // the document (-1: none), and which of its runs
    int q0, q1, k0, k1;
};

// The document and run of a slot. One warp: up to 32 documents a lane each, else 32 candidates a step for the last d with
// q_start[d] / run + d <= slot; the last step has read the starts by the time it knows which it needs.
__device__ __forceinline__ Document find_document(const PkArgs& p, int slot, int run)
{
    const int lane = lane_id();
    int lo = 0, n = p.docs;
    while (true) {
        const int step = (n + 31) / 32;
        const bool in = lane * step < n;
        const int d = lo + (in ? lane * step : 0);
        const int q0 = __ldg(p.q_start + d), q1 = __ldg(p.q_start + d + 1), k0 = __ldg(p.k_start + d), k1 = __ldg(p.k_start + d + 1);
        uint32_t yes;
        int tile;
        if (p.docs <= 32) {
            // Longest first: a document's slots follow those of all with more keys (of as many: with lower numbers). 32 clips of 100 to
            // 1270 rows and 6 heads of 128 take 74 us so and 82 by row number, 32 of 100 rows and 6 heads of 64 12.5 and 14, 5
            // documents of 33024 rows 590 and 600; 32 of 60 rows and 20 heads 28 and 26.5. For more documents than lanes the
            // order would take as many steps for each document as there are.
            const bool rows = in && q0 >= 0 && q1 > q0 && q1 <= p.q_rows;
            const int runs = rows ? (q1 - q0 - 1) / run + 1 : 0, keys = max(k1, p.prefix) - max(k0, p.prefix);
            int before = 0;
            for (int o = 0; o < p.docs; ++o) {
                const int other = __shfl_sync(0xffffffffu, keys, o), more = __shfl_sync(0xffffffffu, runs, o);
                if (other > keys || (other == keys && o < lane))
                    before += more;
            }
            tile = slot - before;
            yes = __ballot_sync(0xffffffffu, tile >= 0 && tile < runs);
        } else {
            tile = slot - (q0 / run + d);
            yes = __ballot_sync(0xffffffffu, in && min(max(q0, 0), p.q_rows) / run + d <= slot);
        }
        const int k = yes ? 31 - __clz(yes) : 0;
        if (!yes || step == 1) {
            Document r;
            r.index = yes ? lo + k : -1;
            r.tile = __shfl_sync(0xffffffffu, tile, k);
            r.q0 = __shfl_sync(0xffffffffu, q0, k), r.q1 = __shfl_sync(0xffffffffu, q1, k);
            r.k0 = __shfl_sync(0xffffffffu, k0, k), r.k1 = __shfl_sync(0xffffffffu, k1, k);
            return r;
        }
        lo += k * step;
        n = min(step, n - k * step);
    }
}

// The run of `run_rows` query rows that a slot is, and the keys that they see.
struct Run {
    int row0, q1;             // query rows [row0, q1) (q1: the document's end)
    int a_end, b0, b_end;     // keys [0, a_end) and [b0, b_end)
    bool any;
};

__device__ __forceinline__ Run run_of(const PkArgs& p, int slot, int run_rows)
{
    const Document doc = find_document(p, slot, run_rows);
    Run r;
    r.row0 = doc.q0 + doc.tile * run_rows, r.q1 = doc.q1;
    r.any = !(doc.index < 0 || doc.q0 < 0 || doc.tile < 0 || r.row0 >= r.q1 || r.q1 > p.q_rows || doc.k0 < 0 || doc.k1 < doc.k0 ||
              doc.k1 > p.k_rows);
    r.a_end = p.prefix;
    r.b0 = max(doc.k0, p.prefix);
    r.b_end = max(doc.k1, r.b0);
    if (r.b0 == p.prefix)
        r.a_end = r.b_end, r.b0 = r.b_end; // the document's keys adjoin the prefix: one run of keys
    return r;
}

// The starts ascend within the tensors; what else they say is told to the caller, and such documents are left out. One CTA, all
// of its threads.
__device__ __forceinline__ void check_starts(const PkArgs& p, int threads)
{
    bool bad = false;
    for (int d = threadIdx.x; d <= p.docs; d += threads) {
        const int a = p.q_start[d], b = p.k_start[d];
        bad |= a < 0 || a > p.q_rows || b < 0 || b > p.k_rows || (d > 0 && (a < p.q_start[d - 1] || b < p.k_start[d - 1]));
    }
    bad = __syncthreads_or(bad);
    if (threadIdx.x == 0) {
        if (p.status)
            *p.status = bad;
        else if (bad)
            record_data_error(kDataStarts);
    }
}

__device__ __forceinline__ void cluster_place(uint32_t& split, uint32_t& part)
{
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(split));
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(part));
}

// How many of a cluster's `most` CTAs share a run of `blocks` key blocks: one for every `least`, so that long documents are
// split further than short ones.
__device__ __forceinline__ uint32_t parts_of(int blocks, int least, uint32_t most)
{
    return min(most, uint32_t(max(1, (blocks + least - 1) / least)));
}

// ------------------------------------------------------------------------------------------------------------
// Small runs, on the warp-wide m16n8k16 MMA. Warp 0 streams 64-key blocks of K and V through a ring (TMA); warps 1..4 have 16
// stacked rows each, with a maximum, a sum and an output of their own:
//   BY_KEYS  few rows (16 / group query rows a run), where the keys' bytes are what counts: a 128-row tile of the tensor core
//            would be nearly empty and, at 1400 clocks for 128 keys, slower than HBM. The warps have the same rows and take
//            16 keys of each block; their parts, and then the cluster's, are joined in a fixed order.
//   by rows  short documents: 64 / group query rows a run, the warps' rows are different ones. A CTA is a fraction of the big
//            kernel's, starts faster, and two fit an SM: 24 documents of 64 rows and keys and 6 heads of 64 take 5.2 us against
//            8.3 and 13.2 by keys, of 128 dims 6.6 against 9.3 and 15.8.
// S (16 x 16 keys) = Q K^T: Q's fragments in registers, K's by ldmatrix; P stays in registers (an MMA's sums are the next
// one's A fragment); O (16 x HD) += P V, V's fragments by ldmatrix.trans. Keys past a block's end get -infinity and V 0.
constexpr int FEW_ROWS = 16, FEW_KEYS = 64, FEW_STAGES = 3, FEW_WARPS = 4, FEW_NT = 32 + 32 * FEW_WARPS, FEW_SPLIT = 16;
constexpr int FEW_LEAST = 16; // blocks that a CTA takes before another one joins it: about 8 us against 7 of starting and joining

template <int HD>
struct FewSmem {
    static constexpr int TL = FEW_KEYS * HD * 2; // a block's K, and its V
    static constexpr int OFF_ML = FEW_STAGES * 2 * TL;              // (max, sum) of the warps' rows, then of the CTA's
    static constexpr int OFF_BAR = OFF_ML + (FEW_WARPS + 1) * FEW_ROWS * 8;
    static constexpr int TOTAL = OFF_BAR + 128 + 1024;
    // the warps' outputs, then the CTA's, over the ring
    static_assert((FEW_WARPS + 1) * FEW_ROWS * HD * 4 <= FEW_STAGES * 2 * TL);
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <bool F16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if constexpr (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int HD, bool F16, bool BY_KEYS>
__global__ void __launch_bounds__(FEW_NT, 2) small_runs_kernel(const __grid_constant__ PkMaps maps, const PkArgs p, const void* q, int64_t q_stride)
{
    using SM = FewSmem<HD>;
    constexpr int TL = SM::TL;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t* smem = smem_raw + (((raw + 1023) & ~1023u) - raw);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + SM::OFF_BAR); // [FEW_STAGES]
    uint64_t* empty = full + FEW_STAGES;                              // [FEW_STAGES]

    const int warp = warp_id(), lane = lane_id();
    uint32_t split, part;
    cluster_place(split, part);
    constexpr int STACK = BY_KEYS ? FEW_ROWS : FEW_ROWS * FEW_WARPS; // stacked rows of a run
    constexpr int SLICES = BY_KEYS ? 1 : FEW_KEYS / 16;              // 16-key slices of a block that a warp takes
    const int item = blockIdx.x / split, kv_head = item % p.kv_heads, run_rows = STACK / p.group;
    if (blockIdx.x == 0)
        check_starts(p, FEW_NT);
    const Run run = run_of(p, item / p.kv_heads, run_rows);
    if (!run.any)
        return;
    const int a_blocks = (run.a_end + FEW_KEYS - 1) / FEW_KEYS;
    const int blocks = a_blocks + (run.b_end - run.b0 + FEW_KEYS - 1) / FEW_KEYS;
    split = BY_KEYS ? parts_of(blocks, FEW_LEAST, split) : 1;
    if (part >= split)
        return; // (a cluster barrier waits for the threads that are left)
    const int per = (blocks + int(split) - 1) / int(split);
    const int first = min(int(part) * per, blocks);
    const int n = min(per, blocks - first);
    auto block_row = [&](int j) { return first + j < a_blocks ? FEW_KEYS * (first + j) : run.b0 + FEW_KEYS * (first + j - a_blocks); };

    if (threadIdx.x == 0) {
        for (int i = 0; i < FEW_STAGES; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], FEW_WARPS);
        }
        fence_barrier_init();
    }
    __syncthreads();

    const int row_a = (BY_KEYS || warp == 0 ? 0 : (warp - 1) * FEW_ROWS) + (lane >> 2); // this thread's stacked rows: and row_a + 8
    const int quad = lane & 3;                                                           // its pair of columns
    // the query row and head of stacked row r; false: none
    auto row_of = [&](int r, int& row, int& head) {
        row = run.row0 + r / p.group, head = kv_head * p.group + r % p.group;
        return r < run_rows * p.group && row < run.q1;
    };
    float o[HD / 8][4];
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < HD / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            o[i][e] = 0.f;
    bool ok = true;

    if (warp == 0) {
        if (lane == 0) {
            int j = 0;
            for (; j < n; ++j) {
                const int s = j % FEW_STAGES;
                if (!mbar_wait(&empty[s], ((j / FEW_STAGES) & 1) ^ 1))
                    break;
                uint8_t* sk = smem + s * 2 * TL;
                const int row = block_row(j);
                mbar_arrive_expect_tx(&full[s], 2 * TL);
#pragma unroll
                for (int hh = 0; hh < HD / 64; ++hh) {
                    tma_load_3d(sk + hh * (FEW_KEYS * 128), &maps.k, &full[s], hh * 64, kv_head, row);
                    tma_load_3d(sk + TL + hh * (FEW_KEYS * 128), &maps.v, &full[s], hh * 64, kv_head, row);
                }
            }
            // Every load lands before the CTA can exit.
            for (int i = max(0, j - FEW_STAGES); i < j; ++i)
                mbar_wait_landed(&full[i % FEW_STAGES], (i / FEW_STAGES) & 1);
        }
    } else {
        uint32_t qf[HD / 16][4];
        {
            int row, head;
            const uint32_t* qa = row_of(row_a, row, head) ? reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(q) + size_t(row) * q_stride + head * HD) : nullptr;
            const uint32_t* qb = row_of(row_a + 8, row, head) ? reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(q) + size_t(row) * q_stride + head * HD) : nullptr;
#pragma unroll
            for (int k = 0; k < HD / 16; ++k) {
                qf[k][0] = qa ? __ldg(qa + k * 8 + quad) : 0, qf[k][2] = qa ? __ldg(qa + k * 8 + 4 + quad) : 0;
                qf[k][1] = qb ? __ldg(qb + k * 8 + quad) : 0, qf[k][3] = qb ? __ldg(qb + k * 8 + 4 + quad) : 0;
            }
        }
        const int key0 = BY_KEYS ? (warp - 1) * 16 : 0; // this warp's first key of a block
        bool idle = false;                              // no row of this warp's is anybody's
        if constexpr (!BY_KEYS)
            idle = row_a - (lane >> 2) >= min(run_rows, run.q1 - run.row0) * p.group;
        // ldmatrix addresses: lane i gives row i % 8 of matrix i / 8. K: matrices (keys 0-7, 8 dims), (keys 0-7, next 8), (keys 8-15,
        // ...), ...; V: (keys 0-7, 8 dims), (keys 8-15, the same), (keys 0-7, next 8), ...
        const int k_row = key0 + (lane >> 4) * 8 + (lane & 7), k_piece = (lane >> 3) & 1;
        const int v_row = key0 + ((lane >> 3) & 1) * 8 + (lane & 7), v_piece = lane >> 4;
        for (int j = 0; j < n; ++j) {
            const int s = j % FEW_STAGES;
            if (!(ok = mbar_wait(&full[s], (j / FEW_STAGES) & 1)))
                break;
            const int keys = (first + j < a_blocks ? run.a_end : run.b_end) - block_row(j) - key0; // this warp's keys, if under its 16 or 64
            if (keys > 0 && !idle) {
                const uint32_t sk = smem_u32(smem + s * 2 * TL), sv = sk + TL;
                float sc[SLICES][2][4];
#pragma unroll
                for (int u = 0; u < SLICES; ++u) {
                    float c[2][2][4] = {}; // [k half][key half]: two chains a sum
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k) {
                        const int piece = (k & 3) * 2 + k_piece;
                        uint32_t b[4];
                        ldmatrix4(b, sk + (k >> 2) * (FEW_KEYS * 128) + (u * 16 + k_row) * 128 + ((piece ^ (k_row & 7)) << 4));
                        mma16816<F16>(c[k & 1][0], qf[k], b[0], b[1]);
                        mma16816<F16>(c[k & 1][1], qf[k], b[2], b[3]);
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int key = u * 16 + h * 8 + quad * 2 + (e & 1);
                            sc[u][h][e] = key < keys ? c[0][h][e] + c[1][h][e] : -INFINITY;
                        }
                }
                float alpha[2];
                bool need = false;
#pragma unroll
                for (int r = 0; r < 2; ++r) { // rows row_a, row_a + 8
                    float mx = -INFINITY;
#pragma unroll
                    for (int u = 0; u < SLICES; ++u)
                        mx = fmaxf(mx, fmaxf(fmaxf(sc[u][0][2 * r], sc[u][0][2 * r + 1]), fmaxf(sc[u][1][2 * r], sc[u][1][2 * r + 1])));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2)) * p.sl2;
                    const bool grow = mx > m[r] + kRescaleThreshold;
                    alpha[r] = grow ? ex2_approx(m[r] - mx) : 1.f;
                    m[r] = grow ? mx : m[r];
                    l[r] *= alpha[r];
                    need |= grow;
                }
                if (__any_sync(0xffffffffu, need)) {
#pragma unroll
                    for (int i = 0; i < HD / 8; ++i)
                        o[i][0] *= alpha[0], o[i][1] *= alpha[0], o[i][2] *= alpha[1], o[i][3] *= alpha[1];
                }
#pragma unroll
                for (int u = 0; u < SLICES; ++u) {
                    if (u * 16 >= keys)
                        break;
                    uint32_t pa[4]; // P rounded to the values' type; the row sums take the unrounded ones
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float sub = m[r] == -INFINITY ? 0.f : m[r];
                        float e[4];
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int x = 0; x < 2; ++x)
                                e[h * 2 + x] = ex2_approx(fmaf(sc[u][h][2 * r + x], p.sl2, -sub));
                        l[r] += (e[0] + e[1]) + (e[2] + e[3]);
                        pa[r] = pack2<F16>(e[0], e[1]), pa[2 + r] = pack2<F16>(e[2], e[3]);
                    }
                    // V's pairs of keys (2 quad, 2 quad + 1) and 8 on: which to keep in a block's last keys
                    uint32_t mask[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int key = u * 16 + h * 8 + quad * 2;
                        mask[h] = (key < keys ? 0xffffu : 0u) | (key + 1 < keys ? 0xffff0000u : 0u);
                    }
#pragma unroll
                    for (int i = 0; i < HD / 16; ++i) {
                        const int piece = (i & 3) * 2 + v_piece;
                        uint32_t b[4];
                        ldmatrix4_trans(b, sv + (i >> 2) * (FEW_KEYS * 128) + (u * 16 + v_row) * 128 + ((piece ^ (v_row & 7)) << 4));
                        mma16816<F16>(o[2 * i], pa, b[0] & mask[0], b[1] & mask[1]);
                        mma16816<F16>(o[2 * i + 1], pa, b[2] & mask[0], b[3] & mask[1]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0)
                mbar_arrive(&empty[s]);
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) { // a row's sum over its four threads
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        }
    }
    if constexpr (!BY_KEYS) {
        if (warp > 0 && ok)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                int row, head;
                if (!row_of(row_a + 8 * r, row, head))
                    continue;
                const float inv = l[r] > 0.f ? 1.f / l[r] : (l[r] == 0.f ? 0.f : l[r]); // as in `store` below
                uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + size_t(row) * p.out_stride + head * HD) + quad;
#pragma unroll
                for (int i = 0; i < HD / 8; ++i)
                    dst[i * 4] = l[r] == 0.f ? 0u : pack2<F16>(o[i][2 * r] * inv, o[i][2 * r + 1] * inv); // (0 times a value may be a NaN)
            }
        return;
    }
    // The parts: (max, sum) and output of every warp's rows, over the ring.
    __syncthreads();
    float2* ml = reinterpret_cast<float2*>(smem + SM::OFF_ML);
    float* out = reinterpret_cast<float*>(smem);
    if (warp > 0) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int at = (warp - 1) * FEW_ROWS + row_a + 8 * r;
            if (quad == 0)
                ml[at] = ok ? make_float2(m[r], l[r]) : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int i = 0; i < HD / 8; ++i)
                *reinterpret_cast<float2*>(out + at * HD + i * 8 + quad * 2) = make_float2(o[i][2 * r], o[i][2 * r + 1]);
        }
    }
    __syncthreads();
    // A warp a row: lane z of `parts` (at most 16) has part z's (max, sum) and gets its weight; returns the rows' (max, sum).
    auto weigh = [&](float2 a, float& w) {
        float mx = a.x;
#pragma unroll
        for (int d = 8; d > 0; d >>= 1)
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        w = a.y == 0.f ? 0.f : ex2_approx(a.x - (mx == -INFINITY ? 0.f : mx));
        float sum = w * a.y;
#pragma unroll
        for (int d = 8; d > 0; d >>= 1)
            sum += __shfl_xor_sync(0xffffffffu, sum, d);
        return make_float2(__shfl_sync(0xffffffffu, mx, 0), __shfl_sync(0xffffffffu, sum, 0));
    };
    const int piece = lane < HD / 4 ? lane : 0;
    auto store = [&](int r, float4 v, float sum) {
        int row, head;
        if (!row_of(r, row, head) || lane >= HD / 4)
            return;
        const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum); // no key (or none above -infinity): 0; a NaN stays one
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + size_t(row) * p.out_stride + head * HD + piece * 4) =
            make_uint2(pack2<F16>(v.x * inv, v.y * inv), pack2<F16>(v.z * inv, v.w * inv));
    };
    const int rows = min(run_rows, run.q1 - run.row0) * p.group;
    for (int r = warp; r < rows; r += FEW_NT / 32) {
        float w;
        const float2 all = weigh(lane < FEW_WARPS ? ml[lane * FEW_ROWS + r] : make_float2(-INFINITY, 0.f), w);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int z = 0; z < FEW_WARPS; ++z) {
            const float wz = __shfl_sync(0xffffffffu, w, z);
            const float4 v = *reinterpret_cast<const float4*>(out + (z * FEW_ROWS + r) * HD + piece * 4);
            if (wz != 0.f) // a part of no weight may hold anything
                acc.x += wz * v.x, acc.y += wz * v.y, acc.z += wz * v.z, acc.w += wz * v.w;
        }
        if (split == 1) {
            store(r, acc, all.y);
        } else {
            if (lane == 0)
                ml[FEW_WARPS * FEW_ROWS + r] = all;
            if (lane < HD / 4)
                *reinterpret_cast<float4*>(out + (FEW_WARPS * FEW_ROWS + r) * HD + piece * 4) = acc;
        }
    }
    if (split > 1) {
        cluster_sync();
        for (int r = int(part) + warp * int(split); r < rows; r += int(split) * (FEW_NT / 32)) {
            float w;
            const float2 all = weigh(lane < int(split) ? ld_cluster2(smem_u32(ml + FEW_WARPS * FEW_ROWS + r), lane) : make_float2(-INFINITY, 0.f), w);
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
            for (int z = 0; z < int(split); ++z) {
                const float wz = __shfl_sync(0xffffffffu, w, z);
                const float4 v = ld_cluster4(smem_u32(out + (FEW_WARPS * FEW_ROWS + r) * HD + piece * 4), z);
                if (wz != 0.f)
                    acc.x += wz * v.x, acc.y += wz * v.y, acc.z += wz * v.z, acc.w += wz * v.w;
            }
            store(r, acc, all.y);
        }
        cluster_sync(); // no CTA leaves while another reads its shared memory
    }
}

// A run as this CTA has it: TWO query tiles, each of which sees every block of the CTA, or one, whose even blocks are "tile"
// 0's and odd ones tile 1's.
template <int HD, bool F16, bool TWO>
__device__ __forceinline__ void attend(const PkMaps& maps, const PkArgs& p, const Run& run, int kv_head, uint32_t split, uint32_t part, int a_blocks,
                                       int blocks)
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
    uint64_t* v_full = k_empty + KST;      // [VST + 1]
    uint64_t* v_empty = v_full + VST + 1;  // [VST + 1]
    uint64_t* s_full = v_empty + VST + 1;  // [2] per tile
    uint64_t* p_full = s_full + 2;     // [2] per tile
    uint64_t* pv_done = p_full + 2;    // [2] per tile
    uint64_t* drain = pv_done + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);

    const int warp = __shfl_sync(0xffffffffu, warp_id(), 0);
    const int row0 = run.row0, q1 = run.q1;
    const int per = (blocks + int(split) - 1) / int(split);
    const int first = min(int(part) * per, blocks);
    const int nkv = min(per, blocks - first); // this CTA's blocks [first, first + nkv)
    // first row and rows of this CTA's block j
    auto block_row = [&](int j) { return first + j < a_blocks ? 128 * (first + j) : run.b0 + 128 * (first + j - a_blocks); };
    auto block_keys = [&](int j) { return min(128, (first + j < a_blocks ? run.a_end : run.b_end) - block_row(j)); };
    constexpr int vst = TWO ? VST : VST + 1;
    // With so few blocks that joining two parts would take longer than it saves, tile 0 has them all.
    const bool alternate = !TWO && (split > 1 || blocks >= 4);
    auto steps = [&](int t) { return TWO ? nkv : alternate ? (nkv + 1 - t) >> 1 : t ? 0 : nkv; }; // of tile t
    auto block_of = [&](int t, int i) { return alternate ? 2 * i + t : i; };                     // its i-th block
    const bool join = split > 1 || alternate; // rows have several parts
    auto k_slot = [&](int j) { return OFF_K + (j % KST) * TL; };
    auto v_slot = [&](int j) { return j % vst < VST ? OFF_V + (j % vst) * TL : TL; };

    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        for (int i = 0; i < KST; ++i) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], 1);
        }
        for (int i = 0; i < VST + 1; ++i) {
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
        const int units = TWO ? 4 : 2;
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
                if (!mbar_wait(&k_empty[jk % KST], ((jk / KST) & 1) ^ 1))
                    break;
                load(smem + k_slot(jk), &maps.k, &k_full[jk % KST], jk);
                ++jk;
            } else {
                if (!mbar_wait(&v_empty[jv % vst], ((jv / vst) & 1) ^ 1))
                    break;
                load(smem + v_slot(jv), &maps.v, &v_full[jv % vst], jv);
                ++jv;
            }
        }
        // Loads that no one waited for (a pipeline that gave up) land before the CTA can exit.
        if (nkv > 0)
            mbar_wait_landed(q_full, 0);
        for (int j = max(0, jk - KST); j < jk; ++j)
            mbar_wait_landed(&k_full[j % KST], (j / KST) & 1);
        for (int j = max(0, jv - vst); j < jv; ++j)
            mbar_wait_landed(&v_full[j % vst], (j / vst) & 1);
    } else if (warp == 1) {
        // ------------------------------------------------------------------------------------------ MMA
        // The warp stays converged and one lane issues, so that descriptors are made in uniform registers.
        uint32_t elected;
        asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(elected));
        const uint32_t id_s = idesc_16<F16>(128, 128, false);
        const uint32_t id_pv = idesc_16<F16>(128, HD, true);
        const uint32_t smem0 = smem_u32(smem);
        // tile t's i-th scores, once their keys are there
        auto scores = [&](int t, int i) {
            const int j = block_of(t, i);
            if (!mbar_wait(&k_full[j % KST], (j / KST) & 1))
                return false;
            tc_fence_after();
            const uint64_t qd = sdesc_sw128(smem0 + (TWO ? t * TL : 0), 16, 1024), kd = sdesc_sw128(smem0 + k_slot(j), 16, 1024);
            if (elected) {
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk) {
                    constexpr int half = HALF >> 4, piece = 32 >> 4;
                    const int off = (kk >> 2) * half + (kk & 3) * piece;
                    mma_bf16_ss(tmem + t * 128, qd + off, kd + off, id_s, kk > 0);
                }
                mma_commit(&s_full[t]);
                if (t == 1 || !TWO)
                    mma_commit(&k_empty[j % KST]); // every tile's S MMAs have read K_j
            }
            __syncwarp();
            return true;
        };
        // its i-th product with V, once P is there
        auto values = [&](int t, int i) {
            const int j = block_of(t, i);
            if (!mbar_wait(&v_full[j % vst], (j / vst) & 1) || !mbar_wait(&p_full[t], i & 1))
                return false;
            tc_fence_after();
            const uint64_t vd = sdesc_sw128(smem0 + v_slot(j), HALF, 1024);
            if (elected) {
#pragma unroll
                for (int kk = 0; kk < 8; ++kk)
                    mma_bf16_ts(tmem + 256 + t * HD, tmem + t * 128 + kk * 8 + (kk >= 4 ? 32 : 0), vd + kk * (2048 >> 4), id_pv, i > 0 || kk > 0);
                mma_commit(&pv_done[t]);
                if (t == 1 || !TWO)
                    mma_commit(&v_empty[j % vst]); // every tile's PV MMAs have read V_j
            }
            __syncwarp();
            return true;
        };
        const int n0 = steps(0), n1 = steps(1);
        bool ok = nkv > 0 && mbar_wait(q_full, 0) && scores(0, 0) && (n1 == 0 || scores(1, 0));
        for (int i = 0; i < n0 && ok; ++i) {
            ok = values(0, i) && (i + 1 >= n0 || scores(0, i + 1));
            if (ok && i < n1)
                ok = values(1, i) && (i + 1 >= n1 || scores(1, i + 1));
        }
        if (elected)
            mma_commit(drain);
        __syncwarp();
        mbar_wait_landed(drain, 0);
    } else if (warp >= 2) {
        // -------------------------------------------------------------------------------------- softmax
        const int t = (warp - 2) / 4;
        const int quarter = warp & 3;
        const int row = quarter * 32 + lane_id();
        const uint32_t lane_base = uint32_t(quarter * 32) << 16;
        const uint32_t tS = tmem + lane_base + t * 128;
        const uint32_t tO = tmem + lane_base + 256 + t * HD;
        // this thread's query row and head
        const int in_unit = row & 63;
        const int out_row = row0 + ((TWO ? 2 * t : 0) + (row >> 6)) * p.unit_rows + in_unit / p.group;
        const bool valid = in_unit < p.unit_rows * p.group && out_row < q1;
        const bool idle = !__any_sync(0xffffffffu, valid); // rows that nobody asked for: their P may be anything
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        const int n = steps(t);
        for (int step = 0; step < n; ++step) {
            if (!(ok = mbar_wait(&s_full[t], step & 1)))
                break;
            tc_fence_after();
            const int j = block_of(t, step);
            const int keys = block_keys(j);
            if (keys < 128 && (t == 0 || !TWO)) {
                // V rows past the block's keys (two tiles: before tile 0's PV, which comes first)
                if (!(ok = mbar_wait(&v_full[j % vst], (j / vst) & 1)))
                    break;
                uint8_t* sv = smem + v_slot(j);
                for (int c = keys * 8 + row; c < 128 * 8; c += 128)
#pragma unroll
                    for (int hh = 0; hh < HD / 64; ++hh)
                        *reinterpret_cast<uint4*>(sv + hh * HALF + c * 16) = make_uint4(0, 0, 0, 0);
                fence_proxy_async_smem();
            }
            if (!idle) {
                // The scores in halves of 64 keys, so that no more than one is in registers: both for the maximum, then the
                // second and the first (read again) for P, which is written over its own half.
                float s[64];
                auto half = [&](int h) {
                    uint32_t r[2][32];
                    tmem_ld32(tS + h * 64, r[0]);
                    tmem_ld32(tS + h * 64 + 32, r[1]);
                    tmem_wait_ld();
#pragma unroll
                    for (int c = 0; c < 64; ++c)
                        s[c] = __uint_as_float(r[c >> 5][c & 31]);
                };
                if (keys < 128)
                    hide_columns(tS, keys);
                float mp[8];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    half(h);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        mp[i] = h ? max3f(mp[i], s[2 * i], s[2 * i + 1]) : fmaxf(s[2 * i], s[2 * i + 1]);
#pragma unroll
                    for (int c = 16; c < 64; c += 16)
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            mp[i] = max3f(mp[i], s[c + 2 * i], s[c + 2 * i + 1]);
                }
                const float mx = max3f(max3f(mp[0], mp[1], mp[2]), max3f(mp[3], mp[4], mp[5]), fmaxf(mp[6], mp[7]));
                const float m_cand = mx * p.sl2;
                const bool need = m_cand > m + kRescaleThreshold;
                const float m_use = need ? m_cand : m;
                const float alpha = need ? ex2_approx(m - m_use) : 1.f;
                const float msub = m_use == -INFINITY ? 0.f : m_use;
                if (step > 0 && __any_sync(0xffffffffu, need)) {
                    // O_t holds the PVs before, complete (these scores were issued after the last of them)
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
                const float2 scale2 = make_float2(p.sl2, p.sl2), neg2 = make_float2(-msub, -msub);
                float2 sp[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int h = 1; h >= 0; --h) {
                    if (h == 0)
                        half(0);
                    uint32_t pk[32]; // P rounded to the values' type for the tensor core; the row sum takes the unrounded ones
#pragma unroll
                    for (int c = 0; c < 32; ++c) {
                        const float2 x = fma2(make_float2(s[2 * c], s[2 * c + 1]), scale2, neg2);
                        const float2 e = make_float2(ex2_approx(x.x), ex2_approx(x.y));
                        sp[c & 3] = add2(sp[c & 3], e);
                        pk[c] = pack2<F16>(e.x, e.y);
                    }
                    tmem_st32(tS + h * 64, pk);
                }
                const float2 s01 = add2(add2(sp[0], sp[1]), add2(sp[2], sp[3]));
                l = l * alpha + (s01.x + s01.y);
                m = m_use;
                tmem_wait_st();
            }
            tc_fence_before();
            __syncwarp();
            if (elect_one_lane())
                mbar_arrive(&p_full[t]);
        }
        const bool done = ok && (n == 0 || mbar_wait(&pv_done[t], (n - 1) & 1));
        if (join) {
            // This part's unnormalised rows and their (max, sum), for the join below, over Q and the rings: the other
            // tile's MMAs must be done with them too. A part that gave up counts for nothing (the device error says so),
            // as one without keys.
            const int other = steps(t ^ 1);
            const bool all = done && (other == 0 || mbar_wait(&pv_done[t ^ 1], (other - 1) & 1)) && n > 0;
            tc_fence_after();
            float* o_row = reinterpret_cast<float*>(smem + OFF_K) + size_t(t * 128 + row) * HD;
            if (!idle) {
                reinterpret_cast<float2*>(smem)[t * 128 + row] = all ? make_float2(m, l) : make_float2(-INFINITY, 0.f);
                if (all) {
#pragma unroll 1
                    for (int c = 0; c < HD / 32; ++c) {
                        uint32_t o[32];
                        tmem_ld32(tO + c * 32, o);
                        tmem_wait_ld();
                        if (valid)
#pragma unroll
                            for (int i = 0; i < 8; ++i) // 16-byte pieces swizzled over the banks
                                *reinterpret_cast<float4*>(o_row + (((c * 8 + i) ^ (row & 7)) << 2)) =
                                    make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]),
                                                __uint_as_float(o[4 * i + 3]));
                    }
                }
            }
        } else if (done && !idle && (TWO || t == 0)) {
            tc_fence_after();
            const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l); // no key (or none above -infinity): 0; a NaN stays one
            uint16_t* dst = static_cast<uint16_t*>(p.out) + size_t(out_row) * p.out_stride + (kv_head * p.group + in_unit % p.group) * HD;
#pragma unroll 1
            for (int c = 0; c < HD / 32; ++c) {
                uint32_t o[32];
                if (n > 0) {
                    tmem_ld32(tO + c * 32, o);
                    tmem_wait_ld();
                }
                if (l == 0.f) // O may hold 0 times an infinity or a NaN
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        o[i] = 0;
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
    if (join) {
        // A warp four rows at a time, whose loads are under way together, the rows dealt out over the cluster's CTAs; parts
        // weighted by 2^(m_part - max), in their order.
        if (split > 1)
            cluster_sync();
        constexpr int AT_ONCE = 4;
        constexpr int tiles = TWO ? 1 : 2, all_rows = TWO ? 256 : 128; // tiles: parts of a row in a CTA
        const int parts = int(split) * tiles, lane = lane_id();
        const int piece = lane < HD / 4 ? lane : 0;
        const int step = int(split) * (NT / 32);
        for (int r0 = int(part) + warp * int(split); r0 < all_rows; r0 += step * AT_ONCE) {
            auto place = [&](int u, int& out_row, int& in_unit) {
                const int r = r0 + u * step;
                in_unit = r & 63;
                out_row = row0 + (r >> 6) * p.unit_rows + in_unit / p.group;
                return r < all_rows && in_unit < p.unit_rows * p.group && out_row < q1;
            };
            float2 a[AT_ONCE]; // lane z: part z's (max, sum), of CTA z / tiles and tile z % tiles
            bool any = false;
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                int out_row, in_unit;
                a[u] = make_float2(-INFINITY, 0.f);
                if (place(u, out_row, in_unit)) {
                    any = true;
                    if (lane < parts)
                        a[u] = ld_cluster2(smem_u32(smem) + (lane % tiles * 128 + r0 + u * step) * 8, lane / tiles);
                }
            }
            if (!any)
                continue;
            float w[AT_ONCE], sum[AT_ONCE];
            float4 acc[AT_ONCE];
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                float mx = a[u].x;
#pragma unroll
                for (int o = 8; o > 0; o >>= 1)
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                w[u] = a[u].y == 0.f ? 0.f : ex2_approx(a[u].x - (mx == -INFINITY ? 0.f : mx));
                sum[u] = w[u] * a[u].y;
#pragma unroll
                for (int o = 8; o > 0; o >>= 1)
                    sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], o);
                sum[u] = __shfl_sync(0xffffffffu, sum[u], 0);
                acc[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll 2
            for (int z = 0; z < parts; ++z)
#pragma unroll
                for (int u = 0; u < AT_ONCE; ++u) {
                    const float wz = __shfl_sync(0xffffffffu, w[u], z);
                    if (wz == 0.f)
                        continue; // a part without keys has written no row, and no row has no part
                    const int at = z % tiles * 128 + r0 + u * step;
                    const float4 v = ld_cluster4(smem_u32(smem + OFF_K) + at * HD * 4 + ((piece ^ (at & 7)) << 4), z / tiles);
                    acc[u].x += wz * v.x, acc[u].y += wz * v.y, acc[u].z += wz * v.z, acc[u].w += wz * v.w;
                }
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                int out_row, in_unit;
                if (!place(u, out_row, in_unit) || lane >= HD / 4)
                    continue;
                const float inv = sum[u] > 0.f ? 1.f / sum[u] : (sum[u] == 0.f ? 0.f : sum[u]);
                uint16_t* dst = static_cast<uint16_t*>(p.out) + size_t(out_row) * p.out_stride + (kv_head * p.group + in_unit % p.group) * HD;
                *reinterpret_cast<uint2*>(dst + piece * 4) =
                    make_uint2(pack2<F16>(acc[u].x * inv, acc[u].y * inv), pack2<F16>(acc[u].z * inv, acc[u].w * inv));
            }
        }
        if (split > 1)
            cluster_sync(); // no CTA leaves while another reads its shared memory
    }
}

template <int HD, bool F16>
__global__ void __launch_bounds__(NT, 1) packed_attention_kernel(const __grid_constant__ PkMaps maps, const PkArgs p)
{
    uint32_t split, part; // CTAs of this run's cluster, this one's number
    cluster_place(split, part);
    if (blockIdx.x == 0)
        check_starts(p, NT);
    const int item = blockIdx.x / split, kv_head = item % p.kv_heads;
    const Run run = run_of(p, item / p.kv_heads, 4 * p.unit_rows);
    if (!run.any)
        return;
    const int a_blocks = (run.a_end + 127) / 128;
    const int blocks = a_blocks + (run.b_end - run.b0 + 127) / 128;
    split = blocks < 2 * LEAST ? 1 : parts_of(blocks, LEAST, split);
    if (part >= split)
        return; // (a cluster barrier waits for the threads that are left)
    if (run.row0 + 2 * p.unit_rows < run.q1)
        attend<HD, F16, true>(maps, p, run, kv_head, split, part, a_blocks, blocks);
    else
        attend<HD, F16, false>(maps, p, run, kv_head, split, part, a_blocks, blocks);
}

CUtensorMap rows_map(const void* base, bool f16, int heads, int rows, int64_t stride, int head_dim, int box_heads, int box_rows)
{
    const uint64_t dims[3] = {uint64_t(head_dim), uint64_t(heads), uint64_t(rows)};
    const uint64_t str[2] = {uint64_t(head_dim) * 2, uint64_t(rows > 1 ? stride : int64_t(heads) * head_dim) * 2};
    const uint32_t box[3] = {64, uint32_t(box_heads), uint32_t(box_rows)};
    return make_tmap(f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, base, dims, str, box);
}

template <int HD, bool F16>
void launch(const PackedAttnParams& p, const PkMaps& maps, const PkArgs& a, cudaStream_t s)
{
    cudaLaunchConfig_t c{};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    c.attrs = at;
    c.numAttrs = 1;
    c.stream = s;
    // Every run of every document has a slot (a document of n rows has at most n / rows + 1 runs).
    auto grid = [&](int rows, int split) {
        const long long ctas = ((long long)p.q_rows / rows + p.docs) * p.kv_heads * split;
        if (ctas > 0x7fffffff)
            throw std::invalid_argument("h3k_attention_packed: more runs of rows than a launch holds");
        at[0].val.clusterDim.x = unsigned(split);
        c.gridDim = dim3(unsigned(ctas));
    };
    enum Kernel { BY_KEYS, BY_ROWS, TILES };
    const int run_rows[3] = {FEW_ROWS / a.group, FEW_ROWS * FEW_WARPS / a.group, 4 * a.unit_rows}; // query rows of a run
    auto shape = [&](Kernel k) {
        c.blockDim = dim3(k == TILES ? NT : FEW_NT);
        c.dynamicSmemBytes = k == TILES ? PkSmem<HD>::TOTAL : FewSmem<HD>::TOTAL;
    };
    auto clusters = [&](Kernel k, int size) { // that the device holds at once
        static ClusterLimits by_keys, by_rows, tiles;
        shape(k);
        return double(k == BY_KEYS   ? by_keys.at_once(small_runs_kernel<HD, F16, true>, c, size)
                      : k == BY_ROWS ? by_rows.at_once(small_runs_kernel<HD, F16, false>, c, size)
                                     : tiles.at_once(packed_attention_kernel<HD, F16>, c, size));
    };
    static std::atomic<uint64_t> opt_in[3], wide;
    smem_opt_in(small_runs_kernel<HD, F16, true>, FewSmem<HD>::TOTAL, opt_in[0]);
    smem_opt_in(small_runs_kernel<HD, F16, false>, FewSmem<HD>::TOTAL, opt_in[1]);
    smem_opt_in(packed_attention_kernel<HD, F16>, PkSmem<HD>::TOTAL, opt_in[2]);
    if (!(wide.load() & device_bit())) {
        H3_CUDA(cudaFuncSetAttribute(small_runs_kernel<HD, F16, true>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        wide.fetch_or(device_bit());
    }

    // The kernel and the CTAs of a run's cluster: the least of what the forms would take, in us, on documents of average length
    // (the longest: UNEVEN times as many keys). A form takes the waves of its runs, and at least its longest run. The constants
    // are fits to 1343 calls (1 to 200 documents of 1 to 200 rows on 40 to 6000 keys, even and uneven, four to ten kinds of heads,
    // each in every form): the form so chosen takes 2.3% longer than the fastest one, in the mean; a rule on rows alone 15%, at
    // worst 91 us for 12.8 (heads of 64, 8 rows of 8 shared heads on 6000 keys). What they know nothing of is one document far longer than
    // the others, which is hardly split: 16 documents of a row, 8 heads, 15 on 40 keys and one on 30000 take 118 us (37 by
    // clusters of eight), 200 of 8 rows of 8 shared heads, 199 on 100 keys and one on 20000, 488 (67 by tiles in clusters of five).
    constexpr double UNEVEN = 1.6;
    constexpr double KEYS_ALONE = HD == 128 ? 0.55 : 0.38, KEYS_FULL = HD == 128 ? 0.7 : 0.55; // 64 keys of a run: alone, in a full device
    constexpr double ROWS_BLOCK = HD == 128 ? 2.4 : 1.3;                                       // 64 keys
    constexpr double TILES_BLOCK = HD == 128 ? 1.1 : 0.9;                                      // 128 keys of the mean run
    const double docs = p.docs, keys = p.prefix + (p.k_rows - p.prefix) / docs, stacked = std::ceil(double(p.q_rows) * a.group / docs);
    auto runs_of = [&](Kernel k) { return docs * p.kv_heads * std::ceil(stacked / (run_rows[k] * a.group)); };
    const double blocks64 = std::ceil(keys / 64), long64 = std::ceil(blocks64 * (p.docs > 1 ? UNEVEN : 1));
    const double blocks128 = std::ceil(keys / 128), long128 = std::ceil(blocks128 * (p.docs > 1 ? UNEVEN : 1));
    auto keys_parts = [&](int split, double blocks) { return std::min<double>(split, std::max(1.0, std::ceil(blocks / FEW_LEAST))); };
    auto by_keys_us = [&](int split) {
        const double at_once = clusters(BY_KEYS, split);
        if (at_once < 1)
            return HUGE_VAL;
        const double runs = runs_of(BY_KEYS), w = runs / at_once, waves = std::max(1.0, (w + std::ceil(w)) / 2), used = keys_parts(split, blocks64);
        const double all = std::ceil(blocks64 / used) * (KEYS_ALONE + (KEYS_FULL - KEYS_ALONE) * std::min(1.0, w)) * waves;
        const double one = std::ceil(long64 / keys_parts(split, long64)) * KEYS_ALONE;
        const double launched = (double(p.q_rows) / run_rows[BY_KEYS] + docs) * p.kv_heads * split; // those without work take time too
        return 6 + 6 * (waves - 1) + std::max(all, one) + (used > 1 ? 2 : 0) + 6 * std::max(0.0, launched - runs * used) / clusters(BY_KEYS, 1);
    };
    auto by_rows_us = [&] {
        const double waves = std::max(1.0, std::ceil(runs_of(BY_ROWS) / clusters(BY_ROWS, 1)));
        return 2.5 + 4.5 * (waves - 1) + blocks64 * ROWS_BLOCK * std::max(waves, p.docs > 1 ? UNEVEN : 1.0);
    };
    auto tiles_parts = [&](int split, double blocks) { return blocks < 2 * LEAST ? 1.0 : std::min<double>(split, std::ceil(blocks / LEAST)); };
    auto tiles_us = [&](int split) {
        const double at_once = clusters(TILES, split), used = tiles_parts(split, blocks128);
        if (at_once < 1)
            return HUGE_VAL;
        const double waves = std::max(1.0, std::ceil(runs_of(TILES) / at_once));
        const double around = 9 + (used > 1 ? 6.5 : 0); // starting, storing, and joining parts
        return std::max((around + std::ceil(blocks128 / used) * TILES_BLOCK) * waves, around + std::ceil(long128 / tiles_parts(split, long128)) * TILES_BLOCK);
    };
    Kernel kernel = TILES;
    int split = 1;
    double least = HUGE_VAL;
    auto consider = [&](Kernel k, int n, double us) {
        if (us < least)
            least = us, kernel = k, split = n;
    };
    if (a.group <= FEW_ROWS)
        for (int n = 1; n == 1 || (n <= FEW_SPLIT && n < 2 * keys_parts(FEW_SPLIT, long64)); n *= 2)
            consider(BY_KEYS, n, by_keys_us(n));
    consider(BY_ROWS, 1, by_rows_us());
    for (int n = 1; n <= tiles_parts(MAX_SPLIT, long128); ++n)
        consider(TILES, n, tiles_us(n));

    grid(run_rows[kernel], split);
    shape(kernel);
    if (kernel == BY_KEYS)
        H3_CUDA(cudaLaunchKernelEx(&c, small_runs_kernel<HD, F16, true>, maps, a, p.q, p.q_stride));
    else if (kernel == BY_ROWS)
        H3_CUDA(cudaLaunchKernelEx(&c, small_runs_kernel<HD, F16, false>, maps, a, p.q, p.q_stride));
    else
        H3_CUDA(cudaLaunchKernelEx(&c, packed_attention_kernel<HD, F16>, maps, a));
}

} // namespace

void attention_packed(const PackedAttnParams& p, cudaStream_t s)
{
    const int group = p.heads / p.kv_heads, unit_rows = 64 / group;
    PkMaps maps;
    maps.q = rows_map(p.q, p.f16, p.heads, p.q_rows, p.q_stride, p.head_dim, group, unit_rows);
    // without key rows there is nothing to describe, and no load is made
    maps.k = p.k_rows > 0 ? rows_map(p.k, p.f16, p.kv_heads, p.k_rows, p.k_stride, p.head_dim, 1, 64) : maps.q;
    maps.v = p.k_rows > 0 ? rows_map(p.v, p.f16, p.kv_heads, p.k_rows, p.v_stride, p.head_dim, 1, 64) : maps.q;
    PkArgs a{};
    a.out = p.out, a.out_stride = p.out_stride, a.q_start = p.q_start, a.k_start = p.k_start, a.status = p.status, a.q_rows = p.q_rows, a.k_rows = p.k_rows;
    a.kv_heads = p.kv_heads, a.docs = p.docs, a.prefix = p.prefix, a.group = group, a.unit_rows = unit_rows;
    a.sl2 = float(double(p.scale) * 1.4426950408889634);
    if (p.head_dim == 128)
        (p.f16 ? launch<128, true> : launch<128, false>)(p, maps, a, s);
    else
        (p.f16 ? launch<64, true> : launch<64, false>)(p, maps, a, s);
}

} // namespace h3
