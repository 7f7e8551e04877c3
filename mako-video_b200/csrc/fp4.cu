// Quantisation of rows to microscaled 4-bit floating point and back (layouts in fp4.cuh).
//
// Both are bound by HBM: the quantiser reads a row once and keeps it in registers while the row's maximum is found (nv
// has a scale a row), the inverse reads half a byte and writes two or four for each value. A thread takes runs of 16
// values: an nv block, or half of an mx block whose two threads exchange their maxima by a shuffle. A run moves as one or
// two 32-byte accesses where rows are so aligned (a 16-byte access at a 32-byte stride costs the L2 twice the requests).
#include "common.hpp"
#include "fp4.cuh"
#include "ptx.cuh"

#include <algorithm>
#include <cuda_fp16.h>

namespace h3 {

namespace {

// 32-byte accesses (32-byte aligned).
__device__ __forceinline__ void load32(uint32_t* w, const void* p)
{
    asm("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p));
}
__device__ __forceinline__ void store32(void* p, const uint32_t* w)
{
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                 "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
        "mul.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

__device__ __forceinline__ float2 mul2_rz(float2 a, float2 b)
{
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
        "mul.rz.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// Sixteen consecutive values of a row, as loaded.
template <Elem T>
struct Run {
    static constexpr int WORDS = T == Elem::f32 ? 16 : 8;
    uint32_t w[WORDS];

    __device__ __forceinline__ void load(const void* row, int c, bool wide)
    {
        const uint8_t* p = static_cast<const uint8_t*>(row) + size_t(c) * (T == Elem::f32 ? 4 : 2);
        if (wide) {
#pragma unroll
            for (int i = 0; i < WORDS; i += 8)
                load32(w + i, p + i * 4);
        } else {
#pragma unroll
            for (int i = 0; i < WORDS; i += 4) {
                const uint4 v = __ldg(reinterpret_cast<const uint4*>(p + i * 4));
                w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
            }
        }
    }
    // The bits of the largest magnitude as fp32, a NaN if there is one (compared as integers, an infinity is larger than every
    // number and a NaN than an infinity).
    __device__ __forceinline__ uint32_t largest() const
    {
        uint32_t m = 0;
        if constexpr (T == Elem::f32) {
#pragma unroll
            for (int i = 0; i < WORDS; ++i)
                m = max(m, w[i] & 0x7fffffffu);
            return m;
        } else {
            if constexpr (T == Elem::bf16) {
                __nv_bfloat162 b = __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[0]));
#pragma unroll
                for (int i = 1; i < WORDS; ++i)
                    b = __hmax2_nan(b, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[i])));
                m = *reinterpret_cast<uint32_t*>(&b);
                return max(m & 0xffffu, m >> 16) << 16;
            } else {
                __half2 b = __habs2(*reinterpret_cast<const __half2*>(&w[0]));
#pragma unroll
                for (int i = 1; i < WORDS; ++i)
                    b = __hmax2_nan(b, __habs2(*reinterpret_cast<const __half2*>(&w[i])));
                m = *reinterpret_cast<uint32_t*>(&b);
                return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(max(m & 0xffffu, m >> 16)))));
            }
        }
    }
    __device__ __forceinline__ float2 pair(int i) const
    {
        if constexpr (T == Elem::f32) {
            return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
        } else if constexpr (T == Elem::bf16) {
            return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
        } else {
            return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        }
    }
};

// Four pairs as e2m1 codes, the first value in the lowest bits; half to even, 6 at most.
__device__ __forceinline__ uint32_t e2m1x8(float2 a, float2 b, float2 c, float2 d)
{
    uint32_t r;
    asm("{\n\t.reg .b8 x, y, z, t;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 x, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 y, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 z, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %8, %7;\n\t"
        "mov.b32 %0, {x, y, z, t};\n\t}"
        : "=r"(r)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y), "f"(d.x), "f"(d.y));
    return r;
}

// x >= 0 as e4m3 (half to even, 448 at most), and back.
__device__ __forceinline__ uint32_t to_e4m3(float x)
{
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(x));
    return r & 0xffu;
}
__device__ __forceinline__ float from_e4m3(uint32_t b)
{
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(b)));
    return __half2float(__ushort_as_half(static_cast<unsigned short>(h & 0xffffu)));
}

// 1 / c rounded to nearest for the 126 positive e4m3 numbers: the approximate reciprocal (within an ulp) and a Newton step.
__device__ __forceinline__ float reciprocal_e4m3(float c)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(c));
    return fmaf(r, fmaf(-c, r, 1.f), r);
}

__device__ __forceinline__ float power_of_two(int e) // -127 <= e <= 127 (2^-127 is subnormal)
{
    return __uint_as_float(e > -127 ? uint32_t(e + 127) << 23 : 0x00400000u);
}

// The scale byte of a block whose largest magnitude has the bits `most`, and the sixteen codes of this thread's run.
// rg: 1 / the row's scale (nv). A block (mx) or row (nv) with an infinity or a NaN has codes 0; its scale says NaN.
template <Elem T, Fp4 F>
__device__ __forceinline__ uint2 encode(const Run<T>& x, uint32_t most, float rg, uint32_t& byte)
{
    float2 q[8];
    if constexpr (F == Fp4::mx) {
        if (most >= 0x7f800000u) {
            byte = 255;
            return make_uint2(0, 0);
        }
        // 2^e with e = floor(log2 most) - 2: the division by it is exact, so the codes are those of the exact quotient
        const int e = max(int(most >> 23) - 127 - 2, -127);
        byte = uint32_t(e + 127);
        const float2 inv = make_float2(power_of_two(-e), power_of_two(-e));
#pragma unroll
        for (int i = 0; i < 8; ++i)
            q[i] = mul2(x.pair(i), inv);
    } else {
        // A quotient rounded to nearest from the divisor's rounded reciprocal: one residual step (Markstein).
        const float m = __uint_as_float(most) * rg;
        const float m6 = m * (1.f / 6.f);
        byte = to_e4m3(fmaf(fmaf(-m6, 6.f, m), 1.f / 6.f, m6));
        const float c = from_e4m3(byte);
        const float inv = c > 0.f ? reciprocal_e4m3(c) : 0.f;
        if constexpr (T == Elem::f32) {
            // the same for the codes: fp32 values come as near to the border of two codes as the quotient's rounding
            const float2 rg2 = make_float2(rg, rg), inv2 = make_float2(inv, inv), nc2 = make_float2(-c, -c);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 s = mul2(x.pair(i), rg2);
                const float2 f = mul2(s, inv2);
                q[i] = fma2(fma2(f, nc2, s), inv2, f);
            }
        } else {
            // x / c has to be exact where it lies on the border t of two codes, where ties go by the code, and on its side of it
            // elsewhere. x = t c: the reciprocal of an e4m3 number rounded to nearest is 1 / c (1 + d) with 0 <= d < 2^-24 (so
            // for all eight significands), and t (1 + d) rounded towards zero is t. Else x / c is 2^-13 or more from t (x has 11 bits at
            // most, t c seven), far more than d and the rounding. (33024 x 13824 in 205 us so, 230 by the residual.)
            float k = inv * rg;
            if (rg > 0x1p118f) { // rows below 2^-107: k could overflow
                k = inv;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    q[i] = mul2(x.pair(i), make_float2(rg, rg));
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    q[i] = x.pair(i);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                q[i] = mul2_rz(q[i], make_float2(k, k));
        }
    }
    return make_uint2(e2m1x8(q[0], q[1], q[2], q[3]), e2m1x8(q[4], q[5], q[6], q[7]));
}

__device__ __forceinline__ size_t scale_at(int row, int block, int tiles)
{
    return (size_t(row >> 7) * tiles + (block >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

struct Packed {
    uint8_t *codes, *scales;
    int K, tiles;
};

// Run c of row r: its codes, and with its neighbours the word of their scales. All lanes of a warp, consecutive runs, a row of
// the tensor's or, with scales of 0, one behind them that fills a scale tile; `in`: the row is the tensor's, `number`: it is finite (nv).
template <Elem T, Fp4 F>
__device__ __forceinline__ void store_run(const Packed& out, int r, int c, bool in, bool number, const Run<T>& a, uint32_t most, float rg)
{
    constexpr int PER = fp4_block(F) / 16; // runs of a block
    if constexpr (F == Fp4::mx)
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1)); // the block's other half (both in the row: K is a multiple of 32)
    uint32_t byte = 0;
    uint2 code = make_uint2(0, 0);
    const bool have = in && c < out.K / 16;
    if (have && number)
        code = encode<T, F>(a, most, rg, byte);
    if (have)
        *reinterpret_cast<uint2*>(out.codes + size_t(r) * (out.K / 2) + size_t(c) * 8) = code;
    // four lanes' (eight for mx) bytes into one word
    uint32_t word = byte << (8 * ((c / PER) & 3));
#pragma unroll
    for (int o = PER; o < 4 * PER; o <<= 1)
        word |= __shfl_xor_sync(0xffffffffu, word, o);
    if (c < out.tiles * 4 * PER && (c & (4 * PER - 1)) == 0)
        *reinterpret_cast<uint32_t*>(out.scales + scale_at(r, c / PER, out.tiles)) = word;
}

// The scale of an nv row whose largest magnitude has the bits `most`: 2^(floor(log2 max) - 10), which makes block scales up to
// 2^11 / 6 = 341.3, under e4m3's 448. Returns its reciprocal; not a number: 0, and a NaN for the scale.
__device__ __forceinline__ float row_scale_of(uint32_t most, float& scale)
{
    const int e = max(int(most >> 23) - 127 - 10, -126);
    const bool number = most < 0x7f800000u;
    scale = number ? power_of_two(e) : __uint_as_float(0x7fffffffu);
    return number ? power_of_two(-e) : 0.f;
}

constexpr int QUANT_RUNS = 2;    // runs of 16 values that a thread keeps: few, so that many threads have loads under way
constexpr int QUANT_THREADS = 512; // of a CTA at most

// blockDim.x = 32 x the warps of a row (RUNS runs a thread; a row of more runs than that is read twice instead of kept), or,
// for SHORT rows of one warp, of as many rows.
// (64 registers a thread: 33024 x 5120 in 67 us for mx; unbounded, with 72, 70.)
template <Elem T, Fp4 F, bool SHORT>
__global__ void __launch_bounds__(QUANT_THREADS, 2) quant_fp4_kernel(const void* x, int64_t ldx, int rows, int K, bool wide, uint8_t* codes,
                                                                  uint8_t* scales, float* row_scale)
{
    constexpr int RUNS = QUANT_RUNS;
    __shared__ uint32_t red[QUANT_THREADS / 32];
    const int r = SHORT ? blockIdx.x * (blockDim.x / 32) + warp_id() : blockIdx.x;
    const int step = SHORT ? 32 : blockDim.x, t = SHORT ? lane_id() : threadIdx.x;
    const int runs = K / 16, tiles = fp4_scale_tiles(K, F);
    const bool in = r < rows;
    const uint8_t* row = static_cast<const uint8_t*>(x) + (in ? size_t(r) * ldx * (T == Elem::f32 ? 4 : 2) : 0);

    Run<T> keep[RUNS];
    uint32_t most[RUNS];
    uint32_t all = 0;
#pragma unroll
    for (int i = 0; i < RUNS; ++i) {
        most[i] = 0;
        if (in && t + i * step < runs)
            keep[i].load(row, (t + i * step) * 16, wide);
    }
#pragma unroll
    for (int i = 0; i < RUNS; ++i)
        if (in && t + i * step < runs) {
            most[i] = keep[i].largest();
            all = max(all, most[i]);
        }
    float rg = 1.f;
    if constexpr (F == Fp4::nv) {
        if (in)
            for (int c = t + RUNS * step; c < runs; c += step) {
                Run<T> a;
                a.load(row, c * 16, wide);
                all = max(all, a.largest());
            }
        all = __reduce_max_sync(0xffffffffu, all);
        if constexpr (!SHORT) {
            if (lane_id() == 0)
                red[warp_id()] = all;
            __syncthreads();
            all = __reduce_max_sync(0xffffffffu, lane_id() < int(blockDim.x) / 32 ? red[lane_id()] : 0);
        }
        float scale;
        rg = row_scale_of(all, scale);
        if (in && t == 0)
            row_scale[r] = scale;
    }
    const bool number = F == Fp4::mx || all < 0x7f800000u;
    // The runs come in whole tiles of four scale bytes (2 runs a byte for mx); the tail's bytes and the rows past the
    // tensor's are 0.
    const int padded = tiles * 4 * fp4_block(F) / 16;
    const Packed out{codes, scales, K, tiles};
#pragma unroll
    for (int i = 0; i < RUNS; ++i)
        if (i * step < padded) // the same for the whole CTA: the shuffles see full warps
            store_run<T, F>(out, r, t + i * step, in, number, keep[i], most[i], rg);
    for (int c0 = RUNS * step; c0 < padded; c0 += step) {
        const int c = c0 + t;
        Run<T> a;
        uint32_t m = 0;
        if (in && c < runs) {
            a.load(row, c * 16, wide);
            m = a.largest();
        }
        store_run<T, F>(out, r, c, in, number, a, m, rg);
    }
}

// Many nv rows of 16-bit values: all threads of a row wait for its last value before they go on, and few rows fit an SM's
// registers. So CTAs walk rows, which bulk copies bring into shared memory one ahead of them, and there are up to four times
// as many CTAs as an SM's threads and shared memory hold (registers hold fewer: 8 of the 10 counted at K = 5120), at different
// places in their rows: 33024 x 5120 in 67 to 70 us (6.3 TB/s) against 84 by the kernel above, x 2048 in 31 against 33, x 13824
// in 205 against 270. (A ring of three rows: 73, 33, 215; as many CTAs as fit: 81 at 5120.)
constexpr int RING = 2; // rows
template <Elem T>
__global__ void __launch_bounds__(QUANT_THREADS, 2) quant_many_rows_kernel(const void* x, int64_t ldx, int rows, int K, uint8_t* codes, uint8_t* scales,
                                                                        float* row_scale)
{
    static_assert(T != Elem::f32);
    constexpr int RUNS = QUANT_RUNS;
    extern __shared__ __align__(128) uint8_t ring[]; // [RING][K] values
    __shared__ uint32_t red[2][QUANT_THREADS / 32];
    __shared__ uint64_t full[RING];
    const int step = blockDim.x, t = threadIdx.x;
    const int runs = K / 16;
    const Packed out{codes, scales, K, fp4_scale_tiles(K, Fp4::nv)};
    const int all_rows = (rows + 127) / 128 * 128; // the rows behind the tensor's have scales of 0
    const uint32_t bytes = uint32_t(K) * 2;
    auto fetch = [&](int64_t r, int turn) {
        if (r < rows) {
            mbar_arrive_expect_tx(&full[turn % RING], bytes);
            bulk_load(ring + (turn % RING) * bytes, static_cast<const uint8_t*>(x) + size_t(r) * ldx * 2, bytes, &full[turn % RING]);
        }
    };
    if (t == 0) {
        for (int i = 0; i < RING; ++i)
            mbar_init(&full[i], 1);
        fence_barrier_init();
        for (int i = 0; i < RING; ++i)
            fetch(int64_t(blockIdx.x) + int64_t(i) * gridDim.x, i);
    }
    __syncthreads();
    int turn = 0;
    for (int64_t r = blockIdx.x; r < all_rows; r += gridDim.x, ++turn) {
        const bool in = r < rows;
        const bool late = in && !mbar_wait(&full[turn % RING], (turn / RING) & 1); // (the device error is set: see below)
        const uint4* row = reinterpret_cast<const uint4*>(ring + (turn % RING) * bytes);
        Run<T> keep[RUNS];
        uint32_t most[RUNS], all = 0;
#pragma unroll
        for (int i = 0; i < RUNS; ++i) {
            most[i] = 0;
            if (in && t + i * step < runs) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint4 v = row[(t + i * step) * 2 + j];
                    keep[i].w[4 * j] = v.x, keep[i].w[4 * j + 1] = v.y, keep[i].w[4 * j + 2] = v.z, keep[i].w[4 * j + 3] = v.w;
                }
                most[i] = keep[i].largest();
                all = max(all, most[i]);
            }
        }
        // A wait that gave up, of whichever thread, ends the CTA: all of it, so that no warp waits at the barrier for one that has
        // left, and not before its copies have landed. (Another kernel's failure ends waits long before their time, so that
        // nothing else says that they have.) It goes with the maxima, as what no magnitude is: a barrier that votes costs 2 to
        // 5% of the call.
        constexpr uint32_t LATE = 0xffffffffu;
        all = __reduce_max_sync(0xffffffffu, late ? LATE : all);
        if (lane_id() == 0)
            red[turn & 1][warp_id()] = all;
        __syncthreads(); // the row is in registers, and the warps' maxima are there
        if (t == 0 && !late)
            fetch(r + int64_t(RING) * gridDim.x, turn);
        all = __reduce_max_sync(0xffffffffu, lane_id() < int(blockDim.x) / 32 ? red[turn & 1][lane_id()] : 0);
        if (all == LATE) {
            if (t == 0)
                for (int i = late ? 0 : 1, end = i + RING; i < end; ++i) // this thread's copies that it has not seen land
                    if (r + int64_t(i) * gridDim.x < rows)
                        mbar_wait_landed(&full[(turn + i) % RING], ((turn + i) / RING) & 1, 100000000ll);
            return;
        }
        float scale;
        const float rg = row_scale_of(all, scale);
        if (in && t == 0)
            row_scale[r] = scale;
#pragma unroll
        for (int i = 0; i < RUNS; ++i)
            if (i * step < out.tiles * 4)
                store_run<T, Fp4::nv>(out, int(r), t + i * step, in, all < 0x7f800000u, keep[i], most[i], rg);
    }
}

// A thread an output run of 16 values.
template <Elem T, Fp4 F>
__global__ void __launch_bounds__(256) dequant_fp4_kernel(const uint8_t* codes, const uint8_t* scales, const float* row_scale, int rows, int K,
                                                          bool wide, void* out, int64_t ldo)
{
    const int runs = K / 16, tiles = fp4_scale_tiles(K, F);
    const size_t id = size_t(blockIdx.x) * 256 + threadIdx.x;
    if (id >= size_t(rows) * runs)
        return;
    const int r = int(id / runs), c = int(id % runs);
    const uint2 code = __ldg(reinterpret_cast<const uint2*>(codes + size_t(r) * (K / 2)) + c);
    const uint32_t byte = __ldg(scales + scale_at(r, F == Fp4::mx ? c / 2 : c, tiles));
    float scale;
    if constexpr (F == Fp4::mx)
        scale = byte == 255 ? __uint_as_float(0x7fffffffu) : power_of_two(int(byte) - 127);
    else
        scale = from_e4m3(byte);
    const float g = row_scale ? __ldg(row_scale + r) : 1.f;
    float v[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        uint32_t h;
        const uint16_t b = uint16_t(((i < 4 ? code.x : code.y) >> (8 * (i & 3))) & 0xffu);
        asm("{\n\t.reg .b8 lo, hi;\n\tmov.b16 {lo, hi}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, lo;\n\t}" : "=r"(h) : "h"(b));
        const float2 f = __half22float2(*reinterpret_cast<__half2*>(&h));
        // code x block scale is exact (2 and 4 bits), so the product with the row's scale is the one rounding in fp32
        const float2 y = mul2(mul2(f, make_float2(scale, scale)), make_float2(g, g));
        v[2 * i] = y.x, v[2 * i + 1] = y.y;
    }
    constexpr int WORDS = Run<T>::WORDS;
    uint32_t w[WORDS];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (T == Elem::f32) {
            w[2 * i] = __float_as_uint(v[2 * i]), w[2 * i + 1] = __float_as_uint(v[2 * i + 1]);
        } else if constexpr (T == Elem::bf16) {
            w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
        } else {
            const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    uint8_t* d = static_cast<uint8_t*>(out) + (size_t(r) * ldo + size_t(c) * 16) * (T == Elem::f32 ? 4 : 2);
    if (wide) {
#pragma unroll
        for (int i = 0; i < WORDS; i += 8)
            store32(d + i * 4, w + i);
    } else {
#pragma unroll
        for (int i = 0; i < WORDS; i += 4)
            *reinterpret_cast<uint4*>(d + i * 4) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
    }
}

// Whether every row starts on a 32-byte boundary.
bool rows_wide(const void* p, int64_t ld, int rows, int size)
{
    return reinterpret_cast<uintptr_t>(p) % 32 == 0 && (rows == 1 || ld * size % 32 == 0);
}

template <Elem T, Fp4 F>
void quant(const void* x, int64_t ldx, int rows, int K, void* codes, void* scales, float* row_scale, cudaStream_t s)
{
    const int runs = K / 16, all_rows = (rows + 127) / 128 * 128;
    const bool wide = rows_wide(x, ldx, rows, T == Elem::f32 ? 4 : 2);
    auto* c = static_cast<uint8_t*>(codes);
    auto* sc = static_cast<uint8_t*>(scales);
    const int warps = (runs + 32 * QUANT_RUNS - 1) / (32 * QUANT_RUNS);
    if constexpr (F == Fp4::nv && T != Elem::f32) {
        const int threads = 32 * warps, held = num_sms() * std::max(1, int(std::min<int64_t>(2048 / threads, 220000 / (int64_t(RING) * K * 2 + 1200))));
        // four rows a CTA at least, and then more CTAs: 4128 x 13824 takes 32 us by two CTAs a place and 37 by four, 4128 x 2048, of
        // one row a CTA, 8.4 against 6.8 by the other kernel
        if (warps > 1 && threads <= QUANT_THREADS && all_rows >= 4 * held) {
            const int ctas = held * std::min(4, all_rows / (4 * held));
            static std::atomic<uint64_t> opt_in;
            smem_opt_in(quant_many_rows_kernel<T>, RING * 32 * QUANT_RUNS * QUANT_THREADS, opt_in);
            quant_many_rows_kernel<T><<<ctas, threads, RING * K * 2, s>>>(x, ldx, rows, K, c, sc, row_scale);
            H3_CUDA(cudaGetLastError());
            return;
        }
    }
    if (warps == 1) // eight rows a CTA
        quant_fp4_kernel<T, F, true><<<all_rows / 8, 256, 0, s>>>(x, ldx, rows, K, wide, c, sc, row_scale);
    else
        quant_fp4_kernel<T, F, false><<<all_rows, std::min(32 * warps, QUANT_THREADS), 0, s>>>(x, ldx, rows, K, wide, c, sc, row_scale);
    H3_CUDA(cudaGetLastError());
}

template <Elem T, Fp4 F>
void dequant(const void* codes, const void* scales, const float* row_scale, int rows, int K, void* out, int64_t ldo, cudaStream_t s)
{
    const size_t n = size_t(rows) * (K / 16);
    dequant_fp4_kernel<T, F><<<unsigned((n + 255) / 256), 256, 0, s>>>(static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales),
                                                                       row_scale, rows, K, rows_wide(out, ldo, rows, T == Elem::f32 ? 4 : 2), out, ldo);
    H3_CUDA(cudaGetLastError());
}

} // namespace

void quant_rows_fp4(const void* x, Elem type, int64_t ldx, int rows, int K, Fp4 f, void* codes, void* scales, float* row_scale,
                    cudaStream_t s)
{
    if (rows <= 0)
        return;
    const bool nv = f == Fp4::nv;
    switch (type) {
    case Elem::bf16: return (nv ? quant<Elem::bf16, Fp4::nv> : quant<Elem::bf16, Fp4::mx>)(x, ldx, rows, K, codes, scales, row_scale, s);
    case Elem::f16: return (nv ? quant<Elem::f16, Fp4::nv> : quant<Elem::f16, Fp4::mx>)(x, ldx, rows, K, codes, scales, row_scale, s);
    case Elem::f32: return (nv ? quant<Elem::f32, Fp4::nv> : quant<Elem::f32, Fp4::mx>)(x, ldx, rows, K, codes, scales, row_scale, s);
    }
}

void dequant_rows_fp4(const void* codes, const void* scales, const float* row_scale, int rows, int K, Fp4 f, Elem type, void* out,
                      int64_t ldo, cudaStream_t s)
{
    if (rows <= 0)
        return;
    const bool nv = f == Fp4::nv;
    switch (type) {
    case Elem::bf16: return (nv ? dequant<Elem::bf16, Fp4::nv> : dequant<Elem::bf16, Fp4::mx>)(codes, scales, row_scale, rows, K, out, ldo, s);
    case Elem::f16: return (nv ? dequant<Elem::f16, Fp4::nv> : dequant<Elem::f16, Fp4::mx>)(codes, scales, row_scale, rows, K, out, ldo, s);
    case Elem::f32: return (nv ? dequant<Elem::f32, Fp4::nv> : dequant<Elem::f32, Fp4::mx>)(codes, scales, row_scale, rows, K, out, ldo, s);
    }
}

} // namespace h3
