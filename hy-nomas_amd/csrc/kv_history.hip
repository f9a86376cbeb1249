// What a long history of the quantized KV cache is kept and read by (gfx950):
//   * bounds of the keys of every block of tokens, channel by channel
//   * the choice of the blocks that a run of queries reads, by those bounds
//   * the choice of the tokens that stay when the cache is cut, by their mass
//   * the move of the kept tokens into another cache
// All stream their operands once or choose among scores that are exact, so that
// the chosen indices do not depend on the order of a sum.
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
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (unit >= a.units) return;  // whole waves; no barrier below
    const int64_t h = unit % a.H, jb = unit / a.H, j = a.j0 + jb % a.blocks, b = jb / a.blocks;
    float lo[16], hi[16];
#pragma unroll
    for (int c = 0; c < 16; ++c) {
        lo[c] = INFINITY;
        hi[c] = -INFINITY;
    }
    const int64_t tok0 = j * a.block;
    const uint8_t* kc = a.kc + b * a.cs0 + h * a.cs2 + piece * 16;
    const float* ks = a.ks + b * a.ss0 + h * a.ss2;
    for (int64_t t0 = tok0; t0 < tok0 + a.block && t0 < a.end; t0 += 64) {
        uint4 x[8];
        float s[8];
        bool ok[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t t = t0 + 8 * i + row;
            ok[i] = t < a.end && (!a.valid || a.valid[b * a.vs + t] != 0);
            if (t < a.end) {
                x[i] = *reinterpret_cast<const uint4*>(kc + t * a.cs1);
                s[i] = ks[t * a.ss1];
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (!ok[i]) continue;
            const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
            for (int c = 0; c < 16; c += 2) {
                const f32x2 f = decode2<FMT>(w[c >> 2], (c >> 1) & 1);
                lo[c] = fminf(lo[c], f[0] * s[i]);
                hi[c] = fmaxf(hi[c], f[0] * s[i]);
                lo[c + 1] = fminf(lo[c + 1], f[1] * s[i]);
                hi[c + 1] = fmaxf(hi[c + 1], f[1] * s[i]);
            }
        }
    }
#pragma unroll
    for (int c = 0; c < 16; ++c)
#pragma unroll
        for (int off = 8; off < 64; off <<= 1) {
            lo[c] = fminf(lo[c], __shfl_xor(lo[c], off, 64));
            hi[c] = fmaxf(hi[c], __shfl_xor(hi[c], off, 64));
        }
    if (row < 2) {  // lanes 0-7 write the lower bounds, lanes 8-15 the upper
        uint32_t w[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const float f0 = row ? hi[2 * c] : lo[2 * c], f1 = row ? hi[2 * c + 1] : lo[2 * c + 1];
            w[c] = f32_to_bf16_bits(f0) | (f32_to_bf16_bits(f1) << 16);
        }
        uint4* dst = reinterpret_cast<uint4*>(a.out + b * a.bs0 + j * a.bs1 + h * a.bs2 + row * D + piece * 16);
        dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
        dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
}

// ---------------------------------------------------------------------------
// Block choice. For a run of queries (its rows over the G query heads of a
// cached head) W_d = sum min(q_d, 0), U_d = sum max(q_d, 0), and
//   score_j = sum_d W_d lo_jd + U_d hi_jd
// bounds the sum of the run's logits with any key of block j. Sums and products
// are in 64 bits: a sum of bf16 values spans far fewer than 53 bits, and so does
// its product with an 8-bit bound, so the score is exact whatever the order of
// its terms (as long as the run's values lie within 2^20 or so of one another)
// and is rounded once, to fp32, to be ranked.

struct PoolArgs {
    const uint16_t* q;
    const uint8_t* qvalid;
    double* pooled;  // [B, Hkv, runs][W 128 | U 128]
    int64_t qs0, qs1, qs2, qvs, Lq, q_block, runs;
    int H, G;
};

__global__ __launch_bounds__(256) void pool_kernel(PoolArgs a) {
    __shared__ double part[4][256];
    const int64_t unit = blockIdx.x;  // (b * H + h) * runs + run
    const int64_t run = unit % a.runs, h = (unit / a.runs) % a.H, b = unit / (a.runs * a.H);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t i0 = run * a.q_block, left = a.Lq - i0;
    const int64_t rows = (left < a.q_block ? left : a.q_block) * a.G;
    double w0 = 0.0, w1 = 0.0, u0 = 0.0, u1 = 0.0;
    for (int64_t r = wave; r < rows; r += 4) {
        const int64_t i = i0 + r / a.G, g = r % a.G;
        if (a.qvalid && a.qvalid[b * a.qvs + i] == 0) continue;
        const uint32_t x = *reinterpret_cast<const uint32_t*>(a.q + b * a.qs0 + i * a.qs1 + (h * a.G + g) * a.qs2 + 2 * lane);
        const float x0 = bf16_lo(x), x1 = bf16_hi(x);
        w0 += x0 > 0.0f ? 0.0f : x0;  // (a NaN enters both sums)
        w1 += x1 > 0.0f ? 0.0f : x1;
        u0 += x0 < 0.0f ? 0.0f : x0;
        u1 += x1 < 0.0f ? 0.0f : x1;
    }
    part[wave][2 * lane] = w0;
    part[wave][2 * lane + 1] = w1;
    part[wave][D + 2 * lane] = u0;
    part[wave][D + 2 * lane + 1] = u1;
    __syncthreads();
    const int t = threadIdx.x;
    a.pooled[unit * 256 + t] = (part[0][t] + part[1][t]) + (part[2][t] + part[3][t]);
}

struct ScoreArgs {
    const double* pooled;
    const uint16_t* bounds;  // [B or 1, blocks, H][lo 128 | hi 128]
    uint32_t* rank;          // [B, H, runs, n]
    int64_t bs0, bs1, bs2, runs, n, first, last;
    int H;
};

HN_DEVICE uint32_t block_rank(const ScoreArgs& a, int64_t j, bool empty, double score) {
    if (empty) return RANK_NONE;
    if (j < a.first || j >= a.n - a.last) return RANK_ALWAYS;
    return rank_of((float)score);
}

// 16 lanes per block, 16 of the 256 terms each.
__global__ __launch_bounds__(256) void score_kernel(ScoreArgs a) {
    const int l16 = threadIdx.x & 15;
    const int64_t j = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    const int64_t bh = blockIdx.y, h = bh % a.H, b = bh / a.H;
    const bool there = j < a.n;
    const uint16_t* src = a.bounds + b * a.bs0 + (there ? j : 0) * a.bs1 + h * a.bs2 + l16 * 16;
    const uint4 x0 = reinterpret_cast<const uint4*>(src)[0], x1 = reinterpret_cast<const uint4*>(src)[1];
    const uint32_t w[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
    const float first = bf16_lo(x0.x);
    const bool empty = __shfl(first, 0, 16) > __shfl(first, 8, 16);
    for (int64_t run = 0; run < a.runs; ++run) {
        const double* p = a.pooled + (bh * a.runs + run) * 256 + l16 * 16;
        double s = 0.0;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            s = __builtin_fma(p[2 * c], (double)bf16_lo(w[c]), s);
            s = __builtin_fma(p[2 * c + 1], (double)bf16_hi(w[c]), s);
        }
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) s += __shfl_xor(s, off, 16);
        if (there && l16 == 0) a.rank[(bh * a.runs + run) * a.n + j] = block_rank(a, j, empty, s);
    }
}

// ---------------------------------------------------------------------------
// The k highest ranks of a row, ties to the lowest index, as ascending indices;
// -1 behind them where fewer can be chosen. A radix search over the rank's four
// digits finds the k-th rank T and how many elements equal to T are taken; each
// wave then writes the chosen indices of its own stretch of the row, from counts
// of the stretches before it.
template <int NT>
struct TopShared {
    uint32_t hist[256];
    uint32_t prefix, need;
    uint32_t above[NT / 64], equal[NT / 64];
};

template <int NT, class Rank>
HN_DEVICE void choose_top(TopShared<NT>& sh, Rank rank, int n, int k, int32_t* out) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    constexpr int WAVES = NT / 64;
    const int kk = k < n ? k : n;
    uint32_t prefix = 0, need = (uint32_t)kk;
    for (int shift = 24; shift >= 0 && kk > 0; shift -= 8) {
        for (int i = tid; i < 256; i += NT) sh.hist[i] = 0;
        __syncthreads();
        for (int i0 = 0; i0 < n; i0 += NT) {
            const int i = i0 + tid;
            const uint32_t u = i < n ? rank(i) : 0u;
            bool in = i < n && (shift == 24 || (u >> (shift + 8)) == (prefix >> (shift + 8)));
            const uint32_t digit = (u >> shift) & 255u;
            if (shift == 24) {
                // most scores share their leading digit: one add per distinct digit of the wave
                while (__any(in)) {
                    const int lead = __builtin_ctzll(__ballot(in));
                    const uint32_t d = __shfl(digit, lead, 64);
                    const uint64_t same = __ballot(in && digit == d);
                    if (lane == lead) atomicAdd(&sh.hist[d], (uint32_t)__builtin_popcountll(same));
                    in = in && digit != d;
                }
            } else if (in) {
                atomicAdd(&sh.hist[digit], 1u);
            }
        }
        __syncthreads();
        if (wave == 0) {  // lane l: bins 4 l .. 4 l + 3
            uint32_t c[4], sum = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += c[e] = sh.hist[4 * lane + e];
            uint32_t suffix = sum;  // of this lane's bins and all above
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
                }
                over += c[e];
            }
        }
        __syncthreads();
        prefix = sh.prefix;
        need = sh.need;
        __syncthreads();  // hist and the two words are rewritten for the next digit
    }
    if (prefix == RANK_NONE) need = 0;
    // the wave's stretch of the row
    const int seg = (((n + WAVES - 1) / WAVES) + 63) / 64 * 64;
    const int lo = wave * seg, hi = lo + seg < n ? lo + seg : n;
    uint32_t above = 0, equal = 0;
    for (int i0 = lo; i0 < hi; i0 += 64) {
        const int i = i0 + lane;
        const uint32_t u = i < hi ? rank(i) : 0u;
        above += (uint32_t)__builtin_popcountll(__ballot(i < hi && u > prefix));
        equal += (uint32_t)__builtin_popcountll(__ballot(i < hi && u == prefix));
    }
    if (lane == 0) {
        sh.above[wave] = above;
        sh.equal[wave] = equal;
    }
    __syncthreads();
    uint32_t pos = 0, eq = 0, total = 0, teq = 0;
    for (int w = 0; w < WAVES; ++w) {
        if (w < wave) {
            pos += sh.above[w];
            eq += sh.equal[w];
        }
        total += sh.above[w];
        teq += sh.equal[w];
    }
    pos += eq < need ? eq : need;
    total += teq < need ? teq : need;
    const uint64_t before = (1ull << lane) - 1;
    if (kk > 0) {
        for (int i0 = lo; i0 < hi; i0 += 64) {
            const int i = i0 + lane;
            const uint32_t u = i < hi ? rank(i) : 0u;
            const uint64_t eqs = __ballot(i < hi && u == prefix);
            const bool take = i < hi && (u > prefix || (u == prefix && eq + (uint32_t)__builtin_popcountll(eqs & before) < need));
            const uint64_t takes = __ballot(take);
            if (take) out[pos + (uint32_t)__builtin_popcountll(takes & before)] = i;
            pos += (uint32_t)__builtin_popcountll(takes);
            eq += (uint32_t)__builtin_popcountll(eqs);
        }
    } else {
        total = 0;
    }
    for (int i = (int)total + tid; i < k; i += NT) out[i] = -1;
}

__global__ __launch_bounds__(256) void choose_blocks_kernel(const uint32_t* __restrict__ rank, int n, int k,
                                                            int32_t* __restrict__ idx) {
    __shared__ TopShared<256> sh;
    const uint32_t* r = rank + (int64_t)blockIdx.x * n;
    choose_top<256>(sh, [&](int i) { return r[i]; }, n, k, idx + (int64_t)blockIdx.x * k);
}

struct TokenArgs {
    const float* mass;
    const uint8_t* valid;
    int32_t* idx;  // [B, H, keep]
    int64_t ms0, ms1, vs;
    int H, n, keep, first, last;
};

__global__ __launch_bounds__(1024) void choose_tokens_kernel(TokenArgs a) {
    __shared__ TopShared<1024> sh;
    const int64_t h = blockIdx.x % a.H, b = blockIdx.x / a.H;
    const float* mass = a.mass + b * a.ms0 + h * a.ms1;
    const uint8_t* valid = a.valid ? a.valid + b * a.vs : nullptr;
    choose_top<1024>(
        sh,
        [&](int i) {
            if (valid && valid[i] == 0) return RANK_NONE;
            if (i < a.first || i >= a.n - a.last) return RANK_ALWAYS;
            return rank_of(mass[i]);
        },
        a.n, a.keep, a.idx + (int64_t)blockIdx.x * a.keep);
}

// ---------------------------------------------------------------------------
// Move of the chosen tokens: row i of the output cache <- row idx[b, h, i] of
// the source (codes and scales of K and V, and the mass), head by head. A
// negative or out-of-range index leaves the row as it is (its mass becomes 0).
struct MoveArgs {
    const uint8_t *k, *v;
    const float *ks, *vs, *mass;
    uint8_t *ok, *ov;
    float *oks, *ovs, *omass;
    const int32_t* idx;
    int64_t cs0, cs1, cs2, ss0, ss1, ss2, ms0, ms1;
    int64_t os0, os1, os2, ts0, ts1, ts2;
    int64_t keep, tokens, rows;
    int H;
};

__global__ __launch_bounds__(256) void move_tokens_kernel(MoveArgs a) {
    const int l = threadIdx.x & 7;
    for (int64_t row = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3); row < a.rows; row += (int64_t)gridDim.x * 32) {
        const int64_t h = row % a.H, i = (row / a.H) % a.keep, b = row / (a.H * a.keep);
        const int64_t at = (b * a.H + h) * a.keep + i;
        const int64_t t = a.idx[at];
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
    HN_REQUIRE(grid <= 0x7fffffffLL, HN_E_ARG, "hn_kv_block_bounds: too many blocks");
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
    HN_REQUIRE(q_block > 0 && top_k > 0 && top_k <= 0x7fffffffLL && blocks <= 0x3fffffffLL, HN_E_ARG,
               "hn_select_kv_blocks: q_block and top_k must be positive");
    HN_REQUIRE(keep_first >= 0 && keep_last >= 0 && keep_first <= top_k && keep_last <= top_k - keep_first, HN_E_ARG,
               "hn_select_kv_blocks: keep_first + keep_last exceeds top_k");
    HN_REQUIRE(qs && bs && qs[3] == 1 && qs[0] % 2 == 0 && qs[1] % 2 == 0 && qs[2] % 2 == 0, HN_E_ARG,
               "hn_select_kv_blocks: q strides");
    HN_REQUIRE(bs[0] % 8 == 0 && bs[1] % 8 == 0 && bs[2] % 8 == 0, HN_E_ARG,
               "hn_select_kv_blocks: bounds strides must be multiples of 8");
    HN_REQUIRE(q_valid_stride >= 0, HN_E_ARG, "hn_select_kv_blocks: negative validity stride");
    HN_REQUIRE(aligned(q, 4) && aligned(bounds, 16) && aligned(idx, 4), HN_E_ARG, "hn_select_kv_blocks: misaligned pointer");
    if (B == 0 || Lq == 0) return HN_OK;
    HN_REQUIRE(q && idx && (bounds || blocks == 0), HN_E_ARG, "hn_select_kv_blocks: null pointer");
    const int64_t runs = (Lq - 1) / q_block + 1;
    const int64_t need = hn_select_kv_blocks_workspace_size(B, H, runs, blocks);
    HN_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned(workspace, 16))), HN_E_ARG,
               "hn_select_kv_blocks: workspace smaller than hn_select_kv_blocks_workspace_size() or misaligned");
    HN_REQUIRE(B * H <= 65535 && B * H * runs <= 0x7fffffffLL, HN_E_ARG, "hn_select_kv_blocks: too much work for one launch");
    if (const int rc = require_gfx950("hn_select_kv_blocks"); rc != HN_OK) return rc;
    hipStream_t st = (hipStream_t)stream;
    uint32_t* rank = nullptr;
    if (blocks > 0) {
        hist::PoolArgs pa;
        pa.q = (const uint16_t*)q; pa.qvalid = q_valid; pa.pooled = (double*)workspace;
        pa.qs0 = qs[0]; pa.qs1 = qs[1]; pa.qs2 = qs[2]; pa.qvs = q_valid_stride;
        pa.Lq = Lq; pa.q_block = q_block; pa.runs = runs; pa.H = (int)H; pa.G = (int)(Hq / H);
        hist::pool_kernel<<<(unsigned)(B * H * runs), 256, 0, st>>>(pa);
        hist::ScoreArgs sa;
        rank = (uint32_t*)((uint8_t*)workspace + align256(B * H * runs * 256 * 8));
        sa.pooled = pa.pooled; sa.bounds = (const uint16_t*)bounds; sa.rank = rank;
        sa.bs0 = bs[0]; sa.bs1 = bs[1]; sa.bs2 = bs[2];
        sa.runs = runs; sa.n = blocks; sa.first = keep_first; sa.last = keep_last; sa.H = (int)H;
        hist::score_kernel<<<dim3((unsigned)((blocks + 15) / 16), (unsigned)(B * H)), 256, 0, st>>>(sa);
    }
    hist::choose_blocks_kernel<<<(unsigned)(B * H * runs), 256, 0, st>>>(rank, (int)blocks, (int)top_k, idx);
    return check_launch("hn_select_kv_blocks");
}

extern "C" int hn_select_kv_tokens(const float* mass, const int64_t* ms, int64_t B, int64_t H, int64_t kv_len,
                                   const uint8_t* valid, int64_t valid_stride, int64_t keep, int64_t keep_first,
                                   int64_t keep_last, int32_t* idx, void* stream) {
    HN_REQUIRE(B >= 0 && H > 0 && kv_len >= 0 && kv_len <= 0x3fffffffLL && keep >= 0 && keep <= 0x3fffffffLL, HN_E_ARG,
               "hn_select_kv_tokens: invalid shape");
    HN_REQUIRE(keep_first >= 0 && keep_last >= 0 && keep_first <= keep && keep_last <= keep - keep_first, HN_E_ARG,
               "hn_select_kv_tokens: keep_first + keep_last exceeds keep");
    HN_REQUIRE(ms && (kv_len < 2 || ms[2] == 1), HN_E_ARG, "hn_select_kv_tokens: the mass of a head must be contiguous");
    HN_REQUIRE(valid_stride >= 0, HN_E_ARG, "hn_select_kv_tokens: negative validity stride");
    HN_REQUIRE(aligned(mass, 4) && aligned(idx, 4), HN_E_ARG, "hn_select_kv_tokens: misaligned pointer");
    if (B == 0 || keep == 0) return HN_OK;
    HN_REQUIRE(idx && (mass || kv_len == 0), HN_E_ARG, "hn_select_kv_tokens: null pointer");
    HN_REQUIRE(B * H <= 0x7fffffffLL, HN_E_ARG, "hn_select_kv_tokens: too many rows");
    if (const int rc = require_gfx950("hn_select_kv_tokens"); rc != HN_OK) return rc;
    hist::TokenArgs a;
    a.mass = mass; a.valid = valid; a.idx = idx;
    a.ms0 = ms[0]; a.ms1 = ms[1]; a.vs = valid_stride;
    a.H = (int)H; a.n = (int)kv_len; a.keep = (int)keep; a.first = (int)keep_first; a.last = (int)keep_last;
    hist::choose_tokens_kernel<<<(unsigned)(B * H), 1024, 0, (hipStream_t)stream>>>(a);
    return check_launch("hn_select_kv_tokens");
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
    HN_REQUIRE(k && v && ks && vs && mass && idx && out_k && out_v && out_ks && out_vs && out_mass, HN_E_ARG,
               "hn_move_kv_tokens: null pointer");
    if (const int rc = require_gfx950("hn_move_kv_tokens"); rc != HN_OK) return rc;
    hist::MoveArgs a;
    a.k = (const uint8_t*)k; a.v = (const uint8_t*)v; a.ks = ks; a.vs = vs; a.mass = mass;
    a.ok = (uint8_t*)out_k; a.ov = (uint8_t*)out_v; a.oks = out_ks; a.ovs = out_vs; a.omass = out_mass; a.idx = idx;
    a.cs0 = cs[0]; a.cs1 = cs[1]; a.cs2 = cs[2]; a.ss0 = ss[0]; a.ss1 = ss[1]; a.ss2 = ss[2];
    a.ms0 = ms[0]; a.ms1 = ms[1];
    a.os0 = os[0]; a.os1 = os[1]; a.os2 = os[2]; a.ts0 = ts[0]; a.ts1 = ts[1]; a.ts2 = ts[2];
    a.keep = keep; a.tokens = tokens; a.rows = B * keep * H; a.H = (int)H;
    const int64_t grid = stream_grid((a.rows + 31) / 32, 16);
    hist::move_tokens_kernel<<<(unsigned)grid, 256, 0, (hipStream_t)stream>>>(a);
    return check_launch("hn_move_kv_tokens");
}
