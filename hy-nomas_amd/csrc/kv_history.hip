// What a long history of the quantized KV cache is kept and read by (gfx950):
//   * bounds of the keys of every block of tokens, channel by channel
//   * the choice of the blocks that a run of queries reads, by those bounds
//   * the choice of the tokens that stay when the cache is cut, by their mass
//   * the move of the kept tokens into another cache
// All stream their operands once; sums have a fixed order, so that the same call gives
// the same indices.
#include "hn_capi_internal.h"
#include "hn_common.h"

namespace hn {
namespace hist {

constexpr int D = 128;

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef double f64x4 __attribute__((ext_vector_type(4)));

// Rank of a score: an unsigned key that is larger for a larger score; -0 ranks
// as +0 and NaN as -inf. The keys of scores lie in [0x007fffff, 0xff800000], so
// RANK_NONE (never chosen) and RANK_ALWAYS lie outside them.
constexpr uint32_t RANK_NONE = 0u, RANK_ALWAYS = 0xffffffffu;

HN_DEVICE uint32_t rank_of(float f) {
    uint32_t u = __float_as_uint(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) u = 0xff800000u;
    if (u == 0x80000000u) u = 0u;
    return (u >> 31) ? ~u : u | 0x80000000u;
}

// ---------------------------------------------------------------------------
// Block bounds: lo = min, hi = max of bf16(code * scale) over a block's valid
// tokens, per channel. Rounding to bf16 is monotone, so the extremes of the
// fp32 products are rounded once at the end. One wave per (batch, block, head):
// 8 lanes hold a key's 128 codes (16 bytes each) and 8 keys are read per load,
// all loads of 64 keys in flight; the 8 keys' extremes meet by lane exchanges.
// Bound by the read of the codes, and for few blocks by the launch: 10800 tokens x 24
// heads (36 MB) 10.4 us, 3.5 TB/s; one token of 8 batches x 8 heads 4.8 us.
struct BoundsArgs {
    const uint8_t* kc;
    const float* ks;
    const uint8_t* valid;
    uint16_t* out;
    int64_t cs0, cs1, cs2, ss0, ss1, ss2, vs, bs0, bs1, bs2;
    int64_t j0, blocks, end, units;
    int H, block;
};

template <int FMT>
HN_DEVICE f32x2 decode2(uint32_t w, int hi) {
    if constexpr (FMT == HN_KV_FP8) {
        return hi ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, 1.0f, true)
                  : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, 1.0f, false);
    } else {
        f32x2 r;
        r[0] = (float)(int8_t)((w >> (16 * hi)) & 0xffu);
        r[1] = (float)(int8_t)((w >> (16 * hi + 8)) & 0xffu);
        return r;
    }
}

template <int FMT>
__global__ __launch_bounds__(256) void bounds_kernel(BoundsArgs a) {
    const int lane = threadIdx.x & 63, piece = lane & 7, row = lane >> 3;
    const uint32_t unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // < 2^31
    if (unit >= a.units) return;  // whole waves; no barrier below
    const uint32_t blocks = (uint32_t)a.blocks, jb = unit / (uint32_t)a.H;
    const int64_t h = unit - jb * (uint32_t)a.H, b = jb / blocks, j = a.j0 + (jb - (uint32_t)b * blocks);
    float lo[16], hi[16];
#pragma unroll
    for (int c = 0; c < 16; ++c) {
        lo[c] = INFINITY;
        hi[c] = -INFINITY;
    }
    const int64_t tok0 = j * a.block;
    const uint32_t code_off = (uint32_t)row * (uint32_t)a.cs1 + 16u * piece, scale_off = (uint32_t)row * (uint32_t)a.ss1 * 4u;
    for (int64_t t0 = tok0; t0 < tok0 + a.block && t0 < a.end; t0 += 64) {
        // descriptors of the 64 keys: rows past the end read as zeros
        const int count = a.end - t0 < 64 ? (int)(a.end - t0) : 64;
        const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint8_t*>(a.kc + b * a.cs0 + t0 * a.cs1 + h * a.cs2), (short)0,
            (int)((count - 1) * a.cs1 + D), 0x00020000);
        const __amdgpu_buffer_rsrc_t sr = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<float*>(a.ks + b * a.ss0 + t0 * a.ss1 + h * a.ss2), (short)0,
            (int)(((count - 1) * a.ss1 + 1) * 4), 0x00020000);
        uint4 x[8];
        float s[8];
        bool ok[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(kr, code_off + 8u * i * (uint32_t)a.cs1, 0, 0));
            s[i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(sr, scale_off + 32u * i * (uint32_t)a.ss1, 0, 0));
            ok[i] = 8 * i + row < count;
        }
        if (a.valid) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (ok[i]) ok[i] = a.valid[b * a.vs + t0 + 8 * i + row] != 0;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
            // a key that does not count becomes NaN, which minimum and maximum pass over
            const float si = ok[i] ? s[i] : __builtin_nanf("");
#pragma unroll
            for (int c = 0; c < 16; c += 2) {
                const f32x2 f = decode2<FMT>(w[c >> 2], (c >> 1) & 1);
                const float p0 = f[0] * si, p1 = f[1] * si;
                lo[c] = fminf(lo[c], p0);
                hi[c] = fmaxf(hi[c], p0);
                lo[c + 1] = fminf(lo[c + 1], p1);
                hi[c + 1] = fmaxf(hi[c + 1], p1);
            }
        }
    }
    // The 8 rows' extremes meet while the channels are dealt out (lane xor 32, 16, 8): each
    // exchange halves a lane's channels, 28 values a lane cross in all where plain
    // reductions would move 96.
    const bool up4 = row & 4, up2 = row & 2, up1 = row & 1;
    float lo8[8], hi8[8], lo4[4], hi4[4], lo2[2], hi2[2];
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        lo8[c] = fminf(up4 ? lo[8 + c] : lo[c], __shfl_xor(up4 ? lo[c] : lo[8 + c], 32, 64));
        hi8[c] = fmaxf(up4 ? hi[8 + c] : hi[c], __shfl_xor(up4 ? hi[c] : hi[8 + c], 32, 64));
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        lo4[c] = fminf(up2 ? lo8[4 + c] : lo8[c], __shfl_xor(up2 ? lo8[c] : lo8[4 + c], 16, 64));
        hi4[c] = fmaxf(up2 ? hi8[4 + c] : hi8[c], __shfl_xor(up2 ? hi8[c] : hi8[4 + c], 16, 64));
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        lo2[c] = fminf(up1 ? lo4[2 + c] : lo4[c], __shfl_xor(up1 ? lo4[c] : lo4[2 + c], 8, 64));
        hi2[c] = fmaxf(up1 ? hi4[2 + c] : hi4[c], __shfl_xor(up1 ? hi4[c] : hi4[2 + c], 8, 64));
    }
    const int c0 = piece * 16 + (up4 ? 8 : 0) + (up2 ? 4 : 0) + (up1 ? 2 : 0);
    uint16_t* dst = a.out + b * a.bs0 + j * a.bs1 + h * a.bs2 + c0;
    *reinterpret_cast<uint32_t*>(dst) = f32_to_bf16_bits(lo2[0]) | (f32_to_bf16_bits(lo2[1]) << 16);
    *reinterpret_cast<uint32_t*>(dst + D) = f32_to_bf16_bits(hi2[0]) | (f32_to_bf16_bits(hi2[1]) << 16);
}

// ---------------------------------------------------------------------------
// Block choice. For a run of queries (its rows over the G query heads of a
// cached head) W_d = sum min(q_d, 0), U_d = sum max(q_d, 0), and
//   score_j = sum_d W_d lo_jd + U_d hi_jd
// bounds the sum of the run's logits with any key of block j. Sums and products
// are in 64 bits and the score is rounded once, to fp32, to be ranked. Where the
// queries' sums (from the highest bit of the largest to the lowest bit of any value in
// them) and the bounds (likewise) span 45 bits together, the 256 products add up exactly,
// whatever their order (values near 1: about 40). Past that a score is off by up to (rows
// + 257) 2^-53 of its terms' magnitudes, in an order that is each kernel's own: the
// kernels for few and for many runs may rank scores apart that differ by no more.

struct PoolArgs {
    const uint16_t* q;
    const uint8_t* qvalid;
    double* pooled;  // [B, Hkv, runs][W 128 | U 128]
    int64_t qs0, qs1, qs2, qvs, Lq, q_block, runs;
    int H, G;
};

HN_DEVICE void add_pooled(uint32_t x, double (&w)[2], double (&u)[2]) {
    const float x0 = bf16_lo(x), x1 = bf16_hi(x);
    w[0] += x0 > 0.0f ? 0.0f : x0;  // (a NaN enters both sums)
    w[1] += x1 > 0.0f ? 0.0f : x1;
    u[0] += x0 < 0.0f ? 0.0f : x0;
    u[1] += x1 < 0.0f ? 0.0f : x1;
}

// One workgroup per run: 16 threads hold a row (8 channels each), 16 rows at a
// time, and the 16 partial sums of a channel meet in LDS. Bound by the read of the
// queries: 10800 x 24 heads (66 MB) 18.6 us, 3.6 TB/s.
__global__ __launch_bounds__(256) void pool_kernel(PoolArgs a) {
    __shared__ double part[16][257];
    const uint32_t unit = blockIdx.x;  // (b * H + h) * runs + run
    const uint32_t runs = (uint32_t)a.runs, bh = unit / runs, H = (uint32_t)a.H, G = (uint32_t)a.G;
    const int64_t run = unit - bh * runs, b = bh / H, h = bh - (uint32_t)b * H;
    const int t = threadIdx.x, l16 = t & 15, g16 = t >> 4;
    const int64_t i0 = run * a.q_block, left = a.Lq - i0;
    const uint32_t rows = (uint32_t)((left < a.q_block ? left : a.q_block) * a.G);  // < 2^31
    double w[4][2] = {}, u[4][2] = {};
    const uint16_t* base = a.q + b * a.qs0 + h * a.G * a.qs2 + 8 * l16;
    for (uint32_t r0 = g16; r0 < rows; r0 += 64) {
        uint4 x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // four rows' loads in flight
            const uint32_t r = r0 + 16 * e, q = r / G, g = r - q * G;
            const int64_t i = i0 + q;
            x[e] = make_uint4(0u, 0u, 0u, 0u);  // adds nothing
            if (r < rows && (!a.qvalid || a.qvalid[b * a.qvs + i] != 0))
                x[e] = *reinterpret_cast<const uint4*>(base + i * a.qs1 + g * a.qs2);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            add_pooled(x[e].x, w[0], u[0]);
            add_pooled(x[e].y, w[1], u[1]);
            add_pooled(x[e].z, w[2], u[2]);
            add_pooled(x[e].w, w[3], u[3]);
        }
    }
    double total = 0.0;
#pragma unroll
    for (int side = 0; side < 2; ++side) {
#pragma unroll
        for (int e = 0; e < 8; ++e) part[g16][8 * l16 + e] = side ? u[e >> 1][e & 1] : w[e >> 1][e & 1];
        __syncthreads();
        if ((t >> 7) == side)
#pragma unroll
            for (int e = 0; e < 16; ++e) total += part[e][t & 127];
        __syncthreads();
    }
    a.pooled[(int64_t)unit * 256 + t] = total;
}

struct ScoreArgs {
    const double* pooled;
    const uint16_t* bounds;  // [B or 1, blocks, H][lo 128 | hi 128]
    uint32_t* rank;          // [B, H, runs, n]
    int64_t bs0, bs1, bs2, runs, n, first, last;
    int H;
    uint32_t run_tiles, stretches, work, per_xcd;  // of score_kernel
    PoolArgs pool;           // the queries, where the kernel sums them itself
};

HN_DEVICE uint32_t block_rank(const ScoreArgs& a, int64_t j, bool empty, double score) {
    if (empty) return RANK_NONE;
    if (j < a.first || j >= a.n - a.last) return RANK_ALWAYS;
    return rank_of((float)score);
}

// Few runs (single tokens): 16 lanes per block, 16 of the 256 terms each, four
// blocks' loads in flight. The run's sums are staged in LDS once per workgroup;
// FROM_Q: they are taken from the queries here (few rows), which saves the pooling
// launch. Bound by the read of the bounds: 64 heads x 2048 blocks (67 MB) 20 us, 3.3
// TB/s.
constexpr int SCORE_FEW_RUNS = 4;
constexpr int SCORE_FEW = 4;  // blocks in flight per lane group
template <bool FROM_Q>
__global__ __launch_bounds__(256, 4) void score_few_kernel(ScoreArgs a) {
    __shared__ __attribute__((aligned(16))) double sums[256];
    const int t = threadIdx.x, l16 = t & 15;
    // heads fastest: the bounds of a block's heads lie side by side
    const int64_t h = blockIdx.x % a.H, b = blockIdx.y, bh = b * a.H + h;
    uint4 x[SCORE_FEW][2];
    int64_t j[SCORE_FEW];
#pragma unroll
    for (int e = 0; e < SCORE_FEW; ++e) {
        j[e] = (int64_t)(blockIdx.x / a.H) * (16 * SCORE_FEW) + 16 * e + (t >> 4);
        const uint4* src = reinterpret_cast<const uint4*>(a.bounds + b * a.bs0 + (j[e] < a.n ? j[e] : 0) * a.bs1 +
                                                          h * a.bs2 + l16 * 16);
        x[e][0] = src[0];
        x[e][1] = src[1];
    }
    for (int64_t run = 0; run < a.runs; ++run) {
        if constexpr (FROM_Q) {
            const PoolArgs& pa = a.pool;
            const int64_t i0 = run * pa.q_block, left = pa.Lq - i0;
            const int rows = (int)((left < pa.q_block ? left : pa.q_block) * pa.G);
            const uint16_t* q = pa.q + b * pa.qs0 + i0 * pa.qs1 + h * pa.G * pa.qs2 + (t & 127);
            double sum = 0.0;
            for (int r0 = 0; r0 < rows; r0 += 4) {
                float y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {  // four rows in flight
                    const int r = r0 + e, i = r / pa.G, g = r % pa.G;
                    y[e] = 0.0f;  // adds nothing
                    if (r < rows && (!pa.qvalid || pa.qvalid[b * pa.qvs + i0 + i] != 0))
                        y[e] = bf16_bits_to_f32(q[i * pa.qs1 + g * pa.qs2]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e)  // threads 0-127 sum min(q, 0), the others max(q, 0); a NaN enters both
                    sum += (t < 128 ? y[e] > 0.0f : y[e] < 0.0f) ? 0.0f : y[e];
            }
            sums[t] = sum;
        } else {
            sums[t] = a.pooled[(bh * a.runs + run) * 256 + t];
        }
        __syncthreads();
        // (the bounds' 64-bit forms are made again for each run: held, they would take
        // four times the registers)
#pragma unroll
        for (int e = 0; e < SCORE_FEW; ++e)
#pragma unroll
            for (int d = 0; d < 2; ++d)
                asm volatile("" : "+v"(x[e][d].x), "+v"(x[e][d].y), "+v"(x[e][d].z), "+v"(x[e][d].w));
        double s[SCORE_FEW] = {};
#pragma unroll
        for (int d = 0; d < 8; ++d) {
            const double2 p = *reinterpret_cast<const double2*>(sums + 16 * l16 + 2 * d);
#pragma unroll
            for (int e = 0; e < SCORE_FEW; ++e) {
                const uint4& z = x[e][d >> 2];
                const uint32_t bits = (d & 3) == 0 ? z.x : (d & 3) == 1 ? z.y : (d & 3) == 2 ? z.z : z.w;
                s[e] = __builtin_fma(p.x, (double)bf16_lo(bits), s[e]);
                s[e] = __builtin_fma(p.y, (double)bf16_hi(bits), s[e]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int e = 0; e < SCORE_FEW; ++e) {
#pragma unroll
            for (int off = 8; off > 0; off >>= 1) s[e] += __shfl_xor(s[e], off, 16);
            const float first = bf16_lo(x[e][0].x);
            const bool empty = __shfl(first, 0, 16) > __shfl(first, 8, 16);
            if (j[e] < a.n && l16 == 0) a.rank[(bh * a.runs + run) * a.n + j[e]] = block_rank(a, j[e], empty, s[e]);
        }
        __syncthreads();  // the sums are rewritten for the next run
    }
}

// Many runs: [runs x 256] x [256 x blocks] on the 64-bit matrix unit, 16 runs x 16
// blocks a wave and v_mfma_f64_16x16x4 (lane l: row or column l % 16, term l / 16;
// result register r: row 4 r + l / 16). Terms are dealt so that lane group g holds
// terms 64 g .. 64 g + 63: each lane then reads 128 contiguous bytes of its block's
// bounds. The runs' sums are staged once per workgroup (row pitch 258 doubles:
// 16-byte reads of 8 rows fall in different banks). Bound by the matrix unit's 64
// cycles a product and by how evenly 864 workgroups fall on 256 CUs: 24 heads x 85 runs
// x 1350 blocks 41 us (1.4 GFLOP, 20 us at the 71 TFLOP/s of a large 64-bit product;
// 48 us with the runs of a stretch of blocks on different XCDs); on the vector unit it
// took 590 us. Two accumulators changed nothing; two tiles a wave took 27 % longer (twice
// the staging).
constexpr int SCORE_TILES = 4;  // 16-block tiles per wave
__global__ __launch_bounds__(256) void score_kernel(ScoreArgs a) {
    constexpr int PITCH = 258;
    __shared__ __attribute__((aligned(16))) double sums[16 * PITCH];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c16 = lane & 15, g = lane >> 4;
    // id % 8 (the XCD) picks a contiguous range of items, the runs of a stretch of blocks
    // side by side: they share its bounds in one L2
    const uint32_t w = (blockIdx.x & 7) * a.per_xcd + (blockIdx.x >> 3);
    if (w >= a.work) return;
    const uint32_t wx = w / a.run_tiles, wz = wx / a.stretches, H = (uint32_t)a.H, wb = wz / H;
    const int64_t bh = wz, h = wz - wb * H, b = wb, run0 = (int64_t)(w - wx * a.run_tiles) * 16;
    const int64_t stretch = wx - wz * a.stretches;
    double in[16];
#pragma unroll
    for (int r = 0; r < 16; ++r)  // (rows past the last run repeat it; their scores are not written)
        in[r] = a.pooled[(bh * a.runs + (run0 + r < a.runs ? run0 + r : a.runs - 1)) * 256 + threadIdx.x];
#pragma unroll
    for (int r = 0; r < 16; ++r) sums[r * PITCH + threadIdx.x] = in[r];
    __syncthreads();
    const double* arow = sums + c16 * PITCH + 64 * g;
    uint4 x[8], y[8];
    auto fetch = [&](int64_t j0) __attribute__((always_inline)) {
        const int64_t j = j0 + c16;
        const uint4* src = reinterpret_cast<const uint4*>(a.bounds + b * a.bs0 + (j < a.n ? j : a.n - 1) * a.bs1 +
                                                          h * a.bs2 + 64 * g);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = src[e];
    };
    const int64_t first_j = (stretch * SCORE_TILES * 4 + wave) * 16;
    fetch(first_j);
    for (int tile = 0; tile < SCORE_TILES; ++tile) {
        const int64_t j0 = first_j + 64 * tile, j = j0 + c16;
        if (j0 >= a.n) break;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = y[e];
        if (tile + 1 < SCORE_TILES) fetch(j0 + 64);  // the next tile's bounds, beside this one's products
        const float first = bf16_lo(x[0].x);
        const bool empty = __shfl(first, c16, 64) > __shfl(first, 32 + c16, 64);
        f64x4 acc = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t w[4] = {x[e].x, x[e].y, x[e].z, x[e].w};
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const double2 s = *reinterpret_cast<const double2*>(arow + 8 * e + 2 * d);
                acc = __builtin_amdgcn_mfma_f64_16x16x4f64(s.x, (double)bf16_lo(w[d]), acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f64_16x16x4f64(s.y, (double)bf16_hi(w[d]), acc, 0, 0, 0);
            }
        }
        if (j < a.n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int64_t run = run0 + 4 * r + g;
                if (run < a.runs) a.rank[(bh * a.runs + run) * a.n + j] = block_rank(a, j, empty, acc[r]);
            }
    }
}

// ---------------------------------------------------------------------------
// The k highest ranks of a row, ties to the lowest index, as ascending indices;
// -1 behind them where fewer can be chosen. One workgroup a row; wave w owns the
// elements [w stretch, (w + 1) stretch). A radix search over the rank's digits, 8
// bits at a time from the top, finds the digits of the k-th rank and how many
// elements that share them are taken; it ends early when all of those are. Each
// wave then writes the chosen indices of its stretch, from counts of the stretches
// before it. Scores share their leading bits, so the digit counts are kept in
// COPIES copies that neighbouring lanes add to. KPT > 0: a thread holds its KPT
// elements in registers (n <= KPT NT), so that a row is read once; KPT = 0: longer
// rows are read again in every pass. Bound by the passes' barriers and LDS adds, not by
// bytes: 2040 rows of 1350 13.6 us, 64 rows of 2048 5.9 us, 24 rows of 1001 masses 8.8
// us, of 32768 23 us.
constexpr int COPIES = 8, COPY_PITCH = 260;  // (a copy starts 4 banks after the one before)

template <int NT>
struct TopShared {
    uint32_t hist[COPIES * COPY_PITCH];
    uint32_t prefix, need, count;
    uint32_t above[NT / 64], equal[NT / 64];
};

// A row's source: load(i) is its raw element (0 past the end: no lane needs a limit),
// rank(i, raw) that element's rank, RANK_NONE past the end.
HN_DEVICE __amdgpu_buffer_rsrc_t row_rsrc(const void* base, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes, 0x00020000);
}

template <int NT, int KPT, class Row>
HN_DEVICE void choose_top(TopShared<NT>& sh, const Row& row, int n, int k, int32_t* out) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    constexpr int WAVES = NT / 64, GROUP = KPT > 0 ? KPT : 8;
    const int stretch = KPT > 0 ? KPT * 64 : (n + NT * GROUP - 1) / (NT * GROUP) * (64 * GROUP);
    const int lo = wave * stretch;
    const int kk = k < n ? k : n;
    uint32_t u[GROUP];
    auto read = [&](int i0) __attribute__((always_inline)) {  // elements i0 + 64 e + lane
#pragma unroll
        for (int e = 0; e < GROUP; ++e) u[e] = row.load(i0 + 64 * e + lane);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = 0; e < GROUP; ++e) {
            u[e] = row.rank(i0 + 64 * e + lane, u[e]);
            if ((e & 3) == 3) __builtin_amdgcn_sched_barrier(0);
        }
    };
    // f(first index, ranks) over the wave's elements, 64 at a time
    auto each = [&](auto f) __attribute__((always_inline)) {
        if constexpr (KPT > 0) {
#pragma unroll
            for (int e = 0; e < GROUP; ++e) {
                f(lo + 64 * e, u[e]);
                if ((e & 3) == 3) __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            for (int i0 = lo; i0 < lo + stretch && i0 < n; i0 += 64 * GROUP) {
                read(i0);
#pragma unroll
                for (int e = 0; e < GROUP; ++e) f(i0 + 64 * e, u[e]);
            }
        }
    };
    if constexpr (KPT > 0) read(lo);
    uint32_t prefix = 0, need = (uint32_t)kk;
    int shift = 32;  // the digits below it are not fixed yet
    while (shift > 0 && kk > 0) {
        shift -= 8;
        for (int i = tid; i < COPIES * COPY_PITCH; i += NT) sh.hist[i] = 0;
        __syncthreads();
        uint32_t* mine = sh.hist + (lane & (COPIES - 1)) * COPY_PITCH;
        each([&](int i0, uint32_t v) __attribute__((always_inline)) {
            if (shift == 24 || ((v ^ prefix) >> (shift + 8)) == 0) atomicAdd(&mine[(v >> shift) & 255u], 1u);
        });
        __syncthreads();
        if (wave == 0) {  // lane l: bins 4 l .. 4 l + 3
            uint32_t c[4] = {0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < COPIES; ++e) {
                const uint4 x = *reinterpret_cast<const uint4*>(sh.hist + e * COPY_PITCH + 4 * lane);
                c[0] += x.x; c[1] += x.y; c[2] += x.z; c[3] += x.w;
            }
            const uint32_t sum = c[0] + c[1] + c[2] + c[3];
            uint32_t suffix = sum;  // of this lane's bins and all above
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const uint32_t o = __shfl_down(suffix, off, 64);
                if (lane + off < 64) suffix += o;
            }
            uint32_t over = suffix - sum;
#pragma unroll
            for (int e = 3; e >= 0; --e) {
                if (over < need && need <= over + c[e]) {
                    sh.prefix = prefix | ((uint32_t)(4 * lane + e) << shift);
                    sh.need = need - over;
                    sh.count = c[e];
                }
                over += c[e];
            }
        }
        __syncthreads();
        prefix = sh.prefix;
        need = sh.need;
        if (sh.count == need) break;  // (every thread reads the same words)
        __syncthreads();  // hist and the words are rewritten for the next digit
    }
    // Taken: ranks whose fixed digits are above prefix's, and the first `need` that
    // equal them (all of them after an early end). RANK_NONE is never taken: it has
    // to be told from the ranks that share its fixed digits.
    uint32_t low = prefix > RANK_NONE ? prefix : 1u, high = shift < 32 ? prefix | ((1u << shift) - 1u) : RANK_ALWAYS;
    uint32_t width = shift < 32 && high >= low ? high - low + 1u : 0u;  // (0: nothing is equal)
    auto is_above = [&](uint32_t v) { return v > high; };
    auto is_equal = [&](uint32_t v) { return v - low < width; };
    uint32_t above = 0, equal = 0;
    each([&](int, uint32_t v) __attribute__((always_inline)) {
        above += is_above(v);
        equal += is_equal(v);
        asm volatile("" : "+v"(above), "+v"(equal));
    });
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        above += __shfl_xor(above, off, 64);
        equal += __shfl_xor(equal, off, 64);
    }
    if (lane == 0) {
        sh.above[wave] = above;
        sh.equal[wave] = equal;
    }
    __syncthreads();
    // counts before this wave's stretch, and of the whole row
    const int w = lane & (WAVES - 1);
    uint32_t total = sh.above[w], teq = sh.equal[w], pos = w < wave ? total : 0u, eq = w < wave ? teq : 0u;
#pragma unroll
    for (int off = WAVES / 2; off > 0; off >>= 1) {
        total += __shfl_xor(total, off, WAVES);
        teq += __shfl_xor(teq, off, WAVES);
        pos += __shfl_xor(pos, off, WAVES);
        eq += __shfl_xor(eq, off, WAVES);
    }
    pos += eq < need ? eq : need;
    total += teq < need ? teq : need;
    const uint64_t before = (1ull << lane) - 1;
    // (the compiler would keep what it knows of every element from the passes before:
    // comparisons as 64-lane masks and indices, more than there are registers)
    int me = lane;
    asm volatile("" : "+v"(low), "+v"(high), "+v"(width), "+v"(me));
    each([&](int i0, uint32_t v) __attribute__((always_inline)) {
        const bool same = is_equal(v);
        const uint64_t eqs = __ballot(same);
        const bool take = is_above(v) || (same && eq + (uint32_t)__builtin_popcountll(eqs & before) < need);
        const uint64_t takes = __ballot(take);
        if (take) out[pos + (uint32_t)__builtin_popcountll(takes & before)] = i0 + me;
        pos += (uint32_t)__builtin_popcountll(takes);
        eq += (uint32_t)__builtin_popcountll(eqs);
        asm volatile("" : "+v"(pos), "+v"(eq));
    });
    for (int i = (int)total + tid; i < k; i += NT) out[i] = -1;
}

struct RankRow {  // ranks as score_kernel wrote them
    __amdgpu_buffer_rsrc_t r;
    HN_DEVICE uint32_t load(int i) const { return __builtin_amdgcn_raw_buffer_load_b32(r, 4 * i, 0, 0); }
    HN_DEVICE uint32_t rank(int, uint32_t raw) const { return raw; }
};

template <int KPT>
__global__ __launch_bounds__(256) void choose_blocks_kernel(const uint32_t* __restrict__ rank, int n, int k,
                                                            int32_t* __restrict__ idx) {
    __shared__ __attribute__((aligned(16))) TopShared<256> sh;
    const RankRow row{row_rsrc(rank + (int64_t)blockIdx.x * n, (int64_t)n * 4)};
    choose_top<256, KPT>(sh, row, n, k, idx + (int64_t)blockIdx.x * k);
}

struct TokenArgs {
    const float* mass;
    const uint8_t* valid;
    int32_t* idx;  // [B, H, keep]
    int64_t ms0, ms1, vs;
    int H, n, keep, first, last;
};

template <bool MASK>
struct MassRow {
    __amdgpu_buffer_rsrc_t m, valid;
    uint32_t n, first, middle;  // tokens [first, first + middle) are ranked by their mass
    HN_DEVICE uint32_t load(int i) const { return __builtin_amdgcn_raw_buffer_load_b32(m, 4 * i, 0, 0); }
    HN_DEVICE uint32_t rank(int i, uint32_t raw) const {
        uint32_t r = rank_of(__uint_as_float(raw));
        if ((uint32_t)i - first >= middle) r = RANK_ALWAYS;
        if (MASK) return __builtin_amdgcn_raw_buffer_load_b8(valid, i, 0, 0) ? r : RANK_NONE;  // (0 past the end)
        return (uint32_t)i < n ? r : RANK_NONE;
    }
};

template <int KPT, bool MASK>
__global__ __launch_bounds__(1024) void choose_tokens_kernel(TokenArgs a) {
    __shared__ __attribute__((aligned(16))) TopShared<1024> sh;
    const int64_t h = blockIdx.x % a.H, b = blockIdx.x / a.H;
    MassRow<MASK> row;
    row.m = row_rsrc(a.mass + b * a.ms0 + h * a.ms1, (int64_t)a.n * 4);
    row.valid = row_rsrc(MASK ? a.valid + b * a.vs : nullptr, MASK ? a.n : 0);
    row.n = (uint32_t)a.n;
    row.first = (uint32_t)a.first;
    row.middle = a.n - a.last > a.first ? (uint32_t)(a.n - a.last - a.first) : 0u;
    choose_top<1024, KPT>(sh, row, a.n, a.keep, a.idx + (int64_t)blockIdx.x * a.keep);
}

// ---------------------------------------------------------------------------
// Token choice in long rows: one workgroup a row leaves most of the device idle, so a
// row is dealt to workgroups of PART tokens and each step of the search is a launch:
// the counts of a digit of the rank (11, 11 and 10 bits) are added to the row's bins
// (whole numbers: the order does not matter), the next launch reads the digit from
// them, the last two count the taken tokens of each part and write them. Bound by its
// six launches: 24 heads x 86400 tokens 37 us, where one workgroup a row took 100 us (a
// row of 32768, the longest that it holds in 74 registers, 23 us).
constexpr int PART_KPT = 16, PART = 256 * PART_KPT, BINS = 2048;

// Per row in the workspace: bins of the three digits, then {prefix, need} after each,
// then {above, equal} of every part.
struct LongRow {
    uint32_t *bins, *state, *counts;
};

HN_DEVICE LongRow long_row(uint32_t* ws, int64_t row, int parts) {
    uint32_t* base = ws + row * (3 * BINS + 8 + 2 * (int64_t)parts);
    return LongRow{base, base + 3 * BINS, base + 3 * BINS + 8};
}

__global__ __launch_bounds__(256) void long_clear_kernel(uint32_t* ws, int parts) {
    const LongRow r = long_row(ws, blockIdx.y, parts);
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < 3 * BINS) r.bins[i] = 0u;
}

// Digit d of a rank lies at bits SHIFT[d] ..; prefix holds the digits before it.
HN_DEVICE constexpr int digit_shift(int d) { return d == 0 ? 21 : d == 1 ? 10 : 0; }
HN_DEVICE constexpr int digit_bins(int d) { return d == 2 ? 1024 : 2048; }

// The digit in which the need-th rank (from the top) lies, from the row's bins of digit
// d: prefix and need move on. Every thread of the 256 gets the same result.
HN_DEVICE void find_digit(const uint32_t* bins, int d, uint32_t& prefix, uint32_t& need, uint32_t* shared) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, per = digit_bins(d) / 256;
    uint32_t c[8], sum = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += c[e] = e < per ? bins[t * per + e] : 0u;
    uint32_t suffix = sum;  // of this thread's bins and all above, in the wave
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t o = __shfl_down(suffix, off, 64);
        if (lane + off < 64) suffix += o;
    }
    if (lane == 0) shared[wave] = suffix;
    __syncthreads();
    uint32_t over = suffix - sum;
    for (int w = wave + 1; w < 4; ++w) over += shared[w];
#pragma unroll
    for (int e = 7; e >= 0; --e) {
        if (over < need && need <= over + c[e]) {
            shared[4] = prefix | ((uint32_t)(t * per + e) << digit_shift(d));
            shared[5] = need - over;
        }
        over += c[e];
    }
    __syncthreads();
    prefix = shared[4];
    need = shared[5];
}

// Launch `step` of the search over a part: 0, 1, 2 count that digit, 3 counts the part's
// taken tokens, 4 writes them.
template <int STEP, bool MASK>
__global__ __launch_bounds__(256) void long_tokens_kernel(TokenArgs a, uint32_t* ws, int parts) {
    __shared__ uint32_t hist[STEP < 3 ? 4 * (BINS + 4) : 4], shared[8], wave_counts[4][2];
    const int64_t rowi = blockIdx.y, h = rowi % a.H, b = rowi / a.H;
    const int part = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const LongRow lr = long_row(ws, rowi, parts);
    MassRow<MASK> row;
    row.m = row_rsrc(a.mass + b * a.ms0 + h * a.ms1, (int64_t)a.n * 4);
    row.valid = row_rsrc(MASK ? a.valid + b * a.vs : nullptr, MASK ? a.n : 0);
    row.n = (uint32_t)a.n;
    row.first = (uint32_t)a.first;
    row.middle = a.n - a.last > a.first ? (uint32_t)(a.n - a.last - a.first) : 0u;
    const int i0 = part * PART + wave * (PART / 4);
    uint32_t u[PART_KPT];
#pragma unroll
    for (int e = 0; e < PART_KPT; ++e) u[e] = row.load(i0 + 64 * e + lane);
    // digits found so far
    uint32_t prefix = 0, need = (uint32_t)(a.keep < a.n ? a.keep : a.n);
    if constexpr (STEP == 2 || STEP == 3) {
        prefix = lr.state[2 * (STEP - 2)];
        need = lr.state[2 * (STEP - 2) + 1];
    }
    if constexpr (STEP >= 1 && STEP <= 3) {
        find_digit(lr.bins + (STEP - 1) * BINS, STEP - 1, prefix, need, shared);
        if (part == 0 && t == 0) {
            lr.state[2 * (STEP - 1)] = prefix;
            lr.state[2 * (STEP - 1) + 1] = need;
        }
    }
    if constexpr (STEP == 4) {
        prefix = lr.state[4];
        need = lr.state[5];
    }
#pragma unroll
    for (int e = 0; e < PART_KPT; ++e) u[e] = row.rank(i0 + 64 * e + lane, u[e]);
    if constexpr (STEP < 3) {
        constexpr int shift = digit_shift(STEP);
        for (int i = t; i < 4 * (BINS + 4); i += 256) hist[i] = 0u;
        __syncthreads();
        uint32_t* mine = hist + (lane & 3) * (BINS + 4);
#pragma unroll
        for (int e = 0; e < PART_KPT; ++e) {
            const bool in = STEP == 0 || ((u[e] ^ prefix) >> digit_shift(STEP > 0 ? STEP - 1 : 0)) == 0;
            if (in) atomicAdd(&mine[(u[e] >> shift) & (uint32_t)(digit_bins(STEP) - 1)], 1u);
        }
        __syncthreads();
        for (int i = t; i < digit_bins(STEP); i += 256) {
            const uint32_t c = hist[i] + hist[BINS + 4 + i] + hist[2 * (BINS + 4) + i] + hist[3 * (BINS + 4) + i];
            if (c) atomicAdd(&lr.bins[STEP * BINS + i], c);
        }
        return;
    }
    // taken: above prefix, and the first `need` equal to it (RANK_NONE, which the bins count
    // too, is never taken: with fewer candidates than places prefix is RANK_NONE)
    uint32_t above = 0, equal = 0;
#pragma unroll
    for (int e = 0; e < PART_KPT; ++e) {
        above += u[e] > prefix;
        equal += u[e] == prefix && u[e] != RANK_NONE;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        above += __shfl_xor(above, off, 64);
        equal += __shfl_xor(equal, off, 64);
    }
    if (lane == 0) {
        wave_counts[wave][0] = above;
        wave_counts[wave][1] = equal;
    }
    __syncthreads();
    if constexpr (STEP == 3) {
        if (t < 2) lr.counts[2 * part + t] = wave_counts[0][t] + wave_counts[1][t] + wave_counts[2][t] + wave_counts[3][t];
        return;
    }
    // counts before this part and of the row, then before this wave
    uint32_t pa = 0, pe = 0, ta = 0, te = 0;
    for (int q = lane; q < parts; q += 64) {
        const uint32_t ca = lr.counts[2 * q], ce = lr.counts[2 * q + 1];
        ta += ca;
        te += ce;
        pa += q < part ? ca : 0u;
        pe += q < part ? ce : 0u;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        pa += __shfl_xor(pa, off, 64);
        pe += __shfl_xor(pe, off, 64);
        ta += __shfl_xor(ta, off, 64);
        te += __shfl_xor(te, off, 64);
    }
    for (int w = 0; w < wave; ++w) {
        pa += wave_counts[w][0];
        pe += wave_counts[w][1];
    }
    uint32_t pos = pa + (pe < need ? pe : need), eq = pe;
    const uint32_t total = ta + (te < need ? te : need);
    int32_t* out = a.idx + rowi * a.keep;
    const uint64_t before = (1ull << lane) - 1;
#pragma unroll
    for (int e = 0; e < PART_KPT; ++e) {
        const bool same = u[e] == prefix && u[e] != RANK_NONE;
        const uint64_t eqs = __ballot(same);
        const bool take = u[e] > prefix || (same && eq + (uint32_t)__builtin_popcountll(eqs & before) < need);
        const uint64_t takes = __ballot(take);
        if (take) out[pos + (uint32_t)__builtin_popcountll(takes & before)] = i0 + 64 * e + lane;
        pos += (uint32_t)__builtin_popcountll(takes);
        eq += (uint32_t)__builtin_popcountll(eqs);
    }
    for (int i = (int)total + part * 256 + t; i < a.keep; i += parts * 256) out[i] = -1;
}

// ---------------------------------------------------------------------------
// Move of the chosen tokens: row i of the output cache <- row idx[b, h, i] of
// the source (codes and scales of K and V, and the mass), head by head. A
// negative or out-of-range index leaves the row as it is (its mass becomes 0). 8 lanes
// move a row. Bound by the scattered 128-byte reads: 43200 of 86400 tokens x 24 heads
// (568 MB) 136 us, 4.2 TB/s (a plain copy reaches 5.1).
struct MoveArgs {
    const uint8_t *k, *v;
    const float *ks, *vs, *mass;
    uint8_t *ok, *ov;
    float *oks, *ovs, *omass;
    const int32_t* idx;
    int64_t cs0, cs1, cs2, ss0, ss1, ss2, ms0, ms1;
    int64_t os0, os1, os2, ts0, ts1, ts2;
    int64_t keep, tokens;
    uint32_t rows, per_xcd;  // of a batch: keep * H, an eighth of it
    int H;
};

__global__ __launch_bounds__(256) void move_tokens_kernel(MoveArgs a) {
    // Workgroup ids are dealt round-robin to the XCDs: id % 8 picks an eighth of the
    // rows, so that the lines of scales and indices that neighbouring rows share are
    // fetched by one L2. (Rows in 32 bits: 64-bit divisions would cost more than the
    // move itself.)
    const int l = threadIdx.x & 7;
    const int64_t b = blockIdx.y;
    const uint32_t H = (uint32_t)a.H, first = (blockIdx.x & 7) * a.per_xcd;
    const uint32_t end = first + a.per_xcd < a.rows ? first + a.per_xcd : a.rows;
    for (uint32_t row = first + (blockIdx.x >> 3) * 32 + (threadIdx.x >> 3); row < end; row += (gridDim.x >> 3) * 32) {
        const uint32_t i = row / H, h = row - i * H;
        const int64_t at = (b * H + h) * a.keep + i;
        const int32_t t = a.idx[at];
        const bool there = t >= 0 && t < a.tokens;
        if (l == 2) a.omass[at] = there ? a.mass[b * a.ms0 + h * a.ms1 + t] : 0.0f;
        if (!there) continue;
        const int64_t from = b * a.cs0 + t * a.cs1 + h * a.cs2 + l * 16, to = b * a.os0 + i * a.os1 + h * a.os2 + l * 16;
        *reinterpret_cast<uint4*>(a.ok + to) = *reinterpret_cast<const uint4*>(a.k + from);
        *reinterpret_cast<uint4*>(a.ov + to) = *reinterpret_cast<const uint4*>(a.v + from);
        const int64_t sf = b * a.ss0 + t * a.ss1 + h * a.ss2, st = b * a.ts0 + i * a.ts1 + h * a.ts2;
        if (l == 0) a.oks[st] = a.ks[sf];
        if (l == 1) a.ovs[st] = a.vs[sf];
    }
}

}  // namespace hist
}  // namespace hn

using namespace hn;

static bool block_size_ok(int64_t block) { return block >= 64 && block <= 1024 && (block & (block - 1)) == 0; }

extern "C" int hn_kv_block_bounds(int fmt, const void* kc, const int64_t* cs, const float* ks, const int64_t* ss,
                                  int64_t B, int64_t H, int64_t D, int64_t cap, int64_t start, int64_t end,
                                  int64_t block, const uint8_t* valid, int64_t valid_stride, void* bounds,
                                  const int64_t* bs, int64_t n_blocks, void* stream) {
    HN_REQUIRE(fmt == HN_KV_FP8 || fmt == HN_KV_INT8, HN_E_ARG, "hn_kv_block_bounds: unknown KV format");
    HN_REQUIRE(D == hist::D, HN_E_ARG, "hn_kv_block_bounds: head dim must be 128");
    HN_REQUIRE(block_size_ok(block), HN_E_ARG, "hn_kv_block_bounds: block must be 64, 128, 256, 512 or 1024");
    HN_REQUIRE(B >= 0 && H > 0 && H <= 65535 && cap >= 0 && start >= 0 && start <= end, HN_E_ARG,
               "hn_kv_block_bounds: invalid shape");
    HN_REQUIRE(end <= cap, HN_E_ARG, "hn_kv_block_bounds: end exceeds the cache capacity");
    HN_REQUIRE((end + block - 1) / block <= n_blocks, HN_E_ARG, "hn_kv_block_bounds: the bounds hold too few blocks");
    HN_REQUIRE(cs && ss && bs, HN_E_ARG, "hn_kv_block_bounds: null stride array");
    HN_REQUIRE(cs[3] == 1 && cs[0] % 16 == 0 && cs[1] % 16 == 0 && cs[2] % 16 == 0, HN_E_ARG,
               "hn_kv_block_bounds: cache strides must be multiples of 16 bytes");
    HN_REQUIRE(cs[1] >= 0 && cs[1] <= 0x1ffffffLL && ss[1] >= 0 && ss[1] <= 0x7fffffLL, HN_E_ARG,
               "hn_kv_block_bounds: invalid cache strides");
    HN_REQUIRE(bs[0] % 8 == 0 && bs[1] % 8 == 0 && bs[2] % 8 == 0, HN_E_ARG,
               "hn_kv_block_bounds: bounds strides must be multiples of 8");
    HN_REQUIRE(valid_stride >= 0, HN_E_ARG, "hn_kv_block_bounds: negative validity stride");
    HN_REQUIRE(aligned(kc, 16) && aligned(bounds, 16) && aligned(ks, 4), HN_E_ARG, "hn_kv_block_bounds: misaligned pointer");
    if (B == 0 || start == end) return HN_OK;
    HN_REQUIRE(kc && ks && bounds, HN_E_ARG, "hn_kv_block_bounds: null pointer");
    if (const int rc = require_gfx950("hn_kv_block_bounds"); rc != HN_OK) return rc;
    hist::BoundsArgs a;
    a.kc = (const uint8_t*)kc; a.ks = ks; a.valid = valid; a.out = (uint16_t*)bounds;
    a.cs0 = cs[0]; a.cs1 = cs[1]; a.cs2 = cs[2];
    a.ss0 = ss[0]; a.ss1 = ss[1]; a.ss2 = ss[2];
    a.bs0 = bs[0]; a.bs1 = bs[1]; a.bs2 = bs[2];
    a.vs = valid_stride;
    a.j0 = start / block;
    a.blocks = (end + block - 1) / block - a.j0;
    a.end = end; a.H = (int)H; a.block = (int)block;
    a.units = B * a.blocks * H;
    const int64_t grid = (a.units + 3) / 4;
    HN_REQUIRE(a.units <= 0x7fffffffLL, HN_E_ARG, "hn_kv_block_bounds: too many blocks");
    hipStream_t st = (hipStream_t)stream;
    if (fmt == HN_KV_FP8) hist::bounds_kernel<HN_KV_FP8><<<(unsigned)grid, 256, 0, st>>>(a);
    else hist::bounds_kernel<HN_KV_INT8><<<(unsigned)grid, 256, 0, st>>>(a);
    return check_launch("hn_kv_block_bounds");
}

static int64_t align256(int64_t n) { return (n + 255) & ~(int64_t)255; }

extern "C" int64_t hn_select_kv_blocks_workspace_size(int64_t B, int64_t H, int64_t runs, int64_t blocks) {
    if (B <= 0 || H <= 0 || runs <= 0 || blocks <= 0) return 0;
    return align256(B * H * runs * 256 * 8) + B * H * runs * blocks * 4;
}

extern "C" int hn_select_kv_blocks(const void* q, const int64_t* qs, int64_t B, int64_t Lq, int64_t Hq, int64_t D,
                                   const uint8_t* q_valid, int64_t q_valid_stride, const void* bounds,
                                   const int64_t* bs, int64_t H, int64_t blocks, int64_t q_block, int64_t top_k,
                                   int64_t keep_first, int64_t keep_last, int32_t* idx, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
    HN_REQUIRE(D == hist::D, HN_E_ARG, "hn_select_kv_blocks: head dim must be 128");
    HN_REQUIRE(B >= 0 && Lq >= 0 && H > 0 && Hq > 0 && Hq % H == 0 && Hq <= 65535 && blocks >= 0, HN_E_ARG,
               "hn_select_kv_blocks: invalid shape");
    HN_REQUIRE(q_block > 0 && top_k > 0, HN_E_ARG, "hn_select_kv_blocks: q_block and top_k must be positive");
    HN_REQUIRE(top_k <= 0x1fffffffLL && blocks <= 0x1fffffffLL, HN_E_ARG, "hn_select_kv_blocks: too many blocks");
    HN_REQUIRE(keep_first >= 0 && keep_last >= 0 && keep_first <= top_k && keep_last <= top_k - keep_first, HN_E_ARG,
               "hn_select_kv_blocks: keep_first + keep_last exceeds top_k");
    HN_REQUIRE(qs && bs && qs[3] == 1 && qs[0] % 8 == 0 && qs[1] % 8 == 0 && qs[2] % 8 == 0, HN_E_ARG,
               "hn_select_kv_blocks: q strides must be multiples of 8");
    HN_REQUIRE(bs[0] % 8 == 0 && bs[1] % 8 == 0 && bs[2] % 8 == 0, HN_E_ARG,
               "hn_select_kv_blocks: bounds strides must be multiples of 8");
    HN_REQUIRE(q_valid_stride >= 0, HN_E_ARG, "hn_select_kv_blocks: negative validity stride");
    HN_REQUIRE(aligned(q, 16) && aligned(bounds, 16) && aligned(idx, 4), HN_E_ARG, "hn_select_kv_blocks: misaligned pointer");
    if (B == 0 || Lq == 0) return HN_OK;
    HN_REQUIRE(q && idx && (bounds || blocks == 0), HN_E_ARG, "hn_select_kv_blocks: null pointer");
    const int64_t runs = (Lq - 1) / q_block + 1;
    const int64_t need = hn_select_kv_blocks_workspace_size(B, H, runs, blocks);
    HN_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned(workspace, 16))), HN_E_ARG,
               "hn_select_kv_blocks: workspace smaller than hn_select_kv_blocks_workspace_size() or misaligned");
    HN_REQUIRE(B * H <= 65535 && B * H * runs <= 0x7fffffffLL && runs <= 16 * 65535LL && Lq <= 0x7fffffffLL / Hq, HN_E_ARG,
               "hn_select_kv_blocks: too much work for one launch");
    if (const int rc = require_gfx950("hn_select_kv_blocks"); rc != HN_OK) return rc;
    hipStream_t st = (hipStream_t)stream;
    uint32_t* rank = nullptr;
    const int64_t rows = B * H * runs, in_run = (q_block < Lq ? q_block : Lq) * (Hq / H);
    if (blocks > 0) {
        hist::PoolArgs pa;
        pa.q = (const uint16_t*)q; pa.qvalid = q_valid; pa.pooled = (double*)workspace;
        pa.qs0 = qs[0]; pa.qs1 = qs[1]; pa.qs2 = qs[2]; pa.qvs = q_valid_stride;
        pa.Lq = Lq; pa.q_block = q_block; pa.runs = runs; pa.H = (int)H; pa.G = (int)(Hq / H);
        hist::ScoreArgs sa = {};
        rank = (uint32_t*)((uint8_t*)workspace + align256(rows * 256 * 8));
        sa.pooled = pa.pooled; sa.bounds = (const uint16_t*)bounds; sa.rank = rank;
        sa.bs0 = bs[0]; sa.bs1 = bs[1]; sa.bs2 = bs[2];
        sa.runs = runs; sa.n = blocks; sa.first = keep_first; sa.last = keep_last; sa.H = (int)H;
        sa.pool = pa;
        const bool few = runs <= hist::SCORE_FEW_RUNS, from_q = few && in_run <= 16;
        if (!from_q) hist::pool_kernel<<<(unsigned)rows, 256, 0, st>>>(pa);
        if (few) {
            constexpr int64_t per = 16 * hist::SCORE_FEW;
            const dim3 grid((unsigned)((blocks + per - 1) / per * H), (unsigned)B);
            if (from_q) hist::score_few_kernel<true><<<grid, 256, 0, st>>>(sa);
            else hist::score_few_kernel<false><<<grid, 256, 0, st>>>(sa);
        } else {
            constexpr int64_t per = 64 * hist::SCORE_TILES;
            const int64_t work = (blocks + per - 1) / per * ((runs + 15) / 16) * B * H;
            HN_REQUIRE(work <= 0x3fffffffLL, HN_E_ARG, "hn_select_kv_blocks: too much work for one launch");
            sa.run_tiles = (uint32_t)((runs + 15) / 16);
            sa.stretches = (uint32_t)((blocks + per - 1) / per);
            sa.work = (uint32_t)work;
            sa.per_xcd = (uint32_t)((work + 7) / 8);
            hist::score_kernel<<<8 * sa.per_xcd, 256, 0, st>>>(sa);
        }
    }
    if (blocks <= 8 * 256)
        hist::choose_blocks_kernel<8><<<(unsigned)rows, 256, 0, st>>>(rank, (int)blocks, (int)top_k, idx);
    else if (blocks <= 32 * 256)
        hist::choose_blocks_kernel<32><<<(unsigned)rows, 256, 0, st>>>(rank, (int)blocks, (int)top_k, idx);
    else
        hist::choose_blocks_kernel<0><<<(unsigned)rows, 256, 0, st>>>(rank, (int)blocks, (int)top_k, idx);
    return check_launch("hn_select_kv_blocks");
}

// Rows of up to this many tokens go to one workgroup each (which then holds them in
// registers), longer ones to several.
constexpr int64_t ONE_GROUP_TOKENS = 32 * 1024;

static int64_t long_parts(int64_t kv_len) { return (kv_len + hist::PART - 1) / hist::PART; }

extern "C" int64_t hn_select_kv_tokens_workspace_size(int64_t B, int64_t H, int64_t kv_len) {
    if (B <= 0 || H <= 0 || kv_len <= ONE_GROUP_TOKENS) return 0;
    return B * H * (3 * hist::BINS + 8 + 2 * long_parts(kv_len)) * (int64_t)sizeof(uint32_t);
}

extern "C" int hn_select_kv_tokens(const float* mass, const int64_t* ms, int64_t B, int64_t H, int64_t kv_len,
                                   const uint8_t* valid, int64_t valid_stride, int64_t keep, int64_t keep_first,
                                   int64_t keep_last, int32_t* idx, void* workspace, int64_t workspace_bytes,
                                   void* stream) {
    HN_REQUIRE(B >= 0 && H > 0 && kv_len >= 0 && kv_len <= 0x1fffffffLL && keep >= 0 && keep <= 0x1fffffffLL, HN_E_ARG,
               "hn_select_kv_tokens: invalid shape");
    HN_REQUIRE(keep_first >= 0 && keep_last >= 0 && keep_first <= keep && keep_last <= keep - keep_first, HN_E_ARG,
               "hn_select_kv_tokens: keep_first + keep_last exceeds keep");
    HN_REQUIRE(ms && (kv_len < 2 || ms[2] == 1), HN_E_ARG, "hn_select_kv_tokens: the mass of a head must be contiguous");
    HN_REQUIRE(valid_stride >= 0, HN_E_ARG, "hn_select_kv_tokens: negative validity stride");
    HN_REQUIRE(aligned(mass, 4) && aligned(idx, 4), HN_E_ARG, "hn_select_kv_tokens: misaligned pointer");
    if (B == 0 || keep == 0) return HN_OK;
    HN_REQUIRE(idx && (mass || kv_len == 0), HN_E_ARG, "hn_select_kv_tokens: null pointer");
    const int64_t need = hn_select_kv_tokens_workspace_size(B, H, kv_len);
    HN_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned(workspace, 16))), HN_E_ARG,
               "hn_select_kv_tokens: workspace smaller than hn_select_kv_tokens_workspace_size() or misaligned");
    HN_REQUIRE(B * H <= 65535, HN_E_ARG, "hn_select_kv_tokens: too many rows");
    if (const int rc = require_gfx950("hn_select_kv_tokens"); rc != HN_OK) return rc;
    hist::TokenArgs a;
    a.mass = mass; a.valid = valid; a.idx = idx;
    a.ms0 = ms[0]; a.ms1 = ms[1]; a.vs = valid_stride;
    a.H = (int)H; a.n = (int)kv_len; a.keep = (int)keep; a.first = (int)keep_first; a.last = (int)keep_last;
    const unsigned grid = (unsigned)(B * H);
    hipStream_t st = (hipStream_t)stream;
    if (kv_len > ONE_GROUP_TOKENS) {
        const int parts = (int)long_parts(kv_len);
        uint32_t* ws = (uint32_t*)workspace;
        const dim3 pg((unsigned)parts, grid);
        hist::long_clear_kernel<<<dim3((3 * hist::BINS + 255) / 256, grid), 256, 0, st>>>(ws, parts);
        if (valid) {
            hist::long_tokens_kernel<0, true><<<pg, 256, 0, st>>>(a, ws, parts);
            hist::long_tokens_kernel<1, true><<<pg, 256, 0, st>>>(a, ws, parts);
            hist::long_tokens_kernel<2, true><<<pg, 256, 0, st>>>(a, ws, parts);
            hist::long_tokens_kernel<3, true><<<pg, 256, 0, st>>>(a, ws, parts);
            hist::long_tokens_kernel<4, true><<<pg, 256, 0, st>>>(a, ws, parts);
        } else {
            hist::long_tokens_kernel<0, false><<<pg, 256, 0, st>>>(a, ws, parts);
            hist::long_tokens_kernel<1, false><<<pg, 256, 0, st>>>(a, ws, parts);
            hist::long_tokens_kernel<2, false><<<pg, 256, 0, st>>>(a, ws, parts);
            hist::long_tokens_kernel<3, false><<<pg, 256, 0, st>>>(a, ws, parts);
            hist::long_tokens_kernel<4, false><<<pg, 256, 0, st>>>(a, ws, parts);
        }
    } else if (kv_len > 8 * 1024) {
        if (valid) hist::choose_tokens_kernel<32, true><<<grid, 1024, 0, st>>>(a);
        else hist::choose_tokens_kernel<32, false><<<grid, 1024, 0, st>>>(a);
    } else {
        if (valid) hist::choose_tokens_kernel<8, true><<<grid, 1024, 0, st>>>(a);
        else hist::choose_tokens_kernel<8, false><<<grid, 1024, 0, st>>>(a);
    }
    return check_launch("hn_select_kv_tokens");
}

// The bytes that a tensor of `n` dims spans from its first element.
struct Span {
    uintptr_t lo, hi;
};

static Span span_of(const void* base, const int64_t* shape, const int64_t* strides, int n, int64_t elem) {
    int64_t last = 0, first = 0;
    for (int i = 0; i < n; ++i) {
        if (shape[i] == 0) return Span{0, 0};
        (strides[i] < 0 ? first : last) += (shape[i] - 1) * strides[i];
    }
    const uintptr_t p = (uintptr_t)base;
    return Span{p + (uintptr_t)(first * elem), p + (uintptr_t)((last + 1) * elem)};
}

extern "C" int hn_move_kv_tokens(const void* k, const void* v, const int64_t* cs, const float* ks, const float* vs,
                                 const int64_t* ss, const float* mass, const int64_t* ms, int64_t B, int64_t H,
                                 int64_t D, int64_t tokens, const int32_t* idx, int64_t keep, void* out_k, void* out_v,
                                 const int64_t* os, float* out_ks, float* out_vs, const int64_t* ts, int64_t out_cap,
                                 float* out_mass, void* stream) {
    HN_REQUIRE(D == hist::D, HN_E_ARG, "hn_move_kv_tokens: head dim must be 128");
    HN_REQUIRE(B >= 0 && H > 0 && H <= 65535 && tokens >= 0 && keep >= 0, HN_E_ARG, "hn_move_kv_tokens: invalid shape");
    HN_REQUIRE(keep <= out_cap, HN_E_ARG, "hn_move_kv_tokens: keep exceeds the output cache's capacity");
    HN_REQUIRE(cs && ss && ms && os && ts, HN_E_ARG, "hn_move_kv_tokens: null stride array");
    HN_REQUIRE(cs[3] == 1 && cs[0] % 16 == 0 && cs[1] % 16 == 0 && cs[2] % 16 == 0 && os[3] == 1 && os[0] % 16 == 0 &&
                   os[1] % 16 == 0 && os[2] % 16 == 0,
               HN_E_ARG, "hn_move_kv_tokens: cache strides must be multiples of 16 bytes");
    HN_REQUIRE(aligned(k, 16) && aligned(v, 16) && aligned(out_k, 16) && aligned(out_v, 16), HN_E_ARG,
               "hn_move_kv_tokens: cache misaligned");
    if (B == 0 || keep == 0) return HN_OK;
    HN_REQUIRE((tokens == 0 || (k && v && ks && vs && mass)) && idx && out_k && out_v && out_ks && out_vs && out_mass,
               HN_E_ARG, "hn_move_kv_tokens: null pointer");
    {
        const int64_t src[4] = {B, tokens, H, D}, dst[4] = {B, keep, H, D}, row[3] = {B, H, tokens};
        const int64_t ms3[3] = {ms[0], ms[1], 1}, flat = B * H * keep, one = 1;
        const Span in[6] = {span_of(k, src, cs, 4, 1), span_of(v, src, cs, 4, 1), span_of(ks, src, ss, 3, 4),
                            span_of(vs, src, ss, 3, 4), span_of(mass, row, ms3, 3, 4), span_of(idx, &flat, &one, 1, 4)};
        const Span out[5] = {span_of(out_k, dst, os, 4, 1), span_of(out_v, dst, os, 4, 1), span_of(out_ks, dst, ts, 3, 4),
                             span_of(out_vs, dst, ts, 3, 4), span_of(out_mass, &flat, &one, 1, 4)};
        for (const Span& o : out)
            for (const Span& i : in)
                HN_REQUIRE(!(o.lo < i.hi && i.lo < o.hi), HN_E_ARG,
                           "hn_move_kv_tokens: the output cache overlaps the source");
    }
    if (const int rc = require_gfx950("hn_move_kv_tokens"); rc != HN_OK) return rc;
    hist::MoveArgs a;
    a.k = (const uint8_t*)k; a.v = (const uint8_t*)v; a.ks = ks; a.vs = vs; a.mass = mass;
    a.ok = (uint8_t*)out_k; a.ov = (uint8_t*)out_v; a.oks = out_ks; a.ovs = out_vs; a.omass = out_mass; a.idx = idx;
    a.cs0 = cs[0]; a.cs1 = cs[1]; a.cs2 = cs[2]; a.ss0 = ss[0]; a.ss1 = ss[1]; a.ss2 = ss[2];
    a.ms0 = ms[0]; a.ms1 = ms[1];
    a.os0 = os[0]; a.os1 = os[1]; a.os2 = os[2]; a.ts0 = ts[0]; a.ts1 = ts[1]; a.ts2 = ts[2];
    HN_REQUIRE(keep * H <= 0x7fffffffLL && B <= 65535, HN_E_ARG, "hn_move_kv_tokens: too many rows for one launch");
    a.keep = keep; a.tokens = tokens; a.rows = (uint32_t)(keep * H); a.H = (int)H;
    a.per_xcd = (a.rows + 255) / 256 * 32;  // whole workgroups of 32 rows
    const int64_t grid = 8 * stream_grid(a.per_xcd / 32, 2);
    hist::move_tokens_kernel<<<dim3((unsigned)grid, (unsigned)B), 256, 0, (hipStream_t)stream>>>(a);
    return check_launch("hn_move_kv_tokens");
}
