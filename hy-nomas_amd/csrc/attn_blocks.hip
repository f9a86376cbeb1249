// Attention over chosen blocks of a quantized KV cache, and the weight that
// each cached key draws (gfx950).
//
//   hn_attn_kv_blocks: O = softmax(Q K^T scale) V and the rows' log-sum-exp, over
//     the keys of the blocks that a list names for each run of queries (without a
//     list: every cached key), then the bf16 tail.
//   hn_attn_key_mass:  mass[t] = sum over query rows of exp(s(row, t) - lse(row)).
//
// K, V = bf16(code * scale), as in attn_fp8kv.hip.
#include "attn_tiles.h"

namespace hn {
namespace attn {

// ---------------------------------------------------------------------------
// Attention over listed blocks: the two-stage loop of attn_fp8kv.hip (4 waves,
// 128 rows, half-tile steps), its cache tiles taken from the list. The rows of a
// workgroup belong to one run of queries and one cached head, so that one list
// serves them all: row r of a run is query r / G and query head r % G of the
// head's group. The part of a tile past kv_len, an entry past the last block and
// invalid keys are masked by the tile's 64-bit word; the V codes and scales of
// masked keys enter LDS as zeros, so that nothing they hold (an unwritten row, an
// Inf or NaN) meets a zero probability.
struct BlockParams : Params {
    const int32_t* idx;    // null: all blocks
    int64_t is0, is1, is2;
    int top_k, shift;      // block = 64 << shift tokens
    int64_t block;
    int64_t q_block, runs, B;
    int G;                 // query heads per cached head; H counts cached heads
    float* lse;            // [B, H G, Lq]
};

// Entries of a list before its first negative one. Every wave counts for itself.
HN_DEVICE int list_length(const int32_t* list, int k) {
    const int lane = threadIdx.x & 63;
    for (int i0 = 0; i0 < k; i0 += 64) {
        const uint64_t end = __ballot(i0 + lane >= k || list[i0 + lane] < 0);
        if (end) return i0 + __builtin_ctzll(end);
    }
    return k;
}

// Step A with the denominator summed from the fp32 probabilities, so that the
// row's log-sum-exp carries no rounding of the fp16 ones (their sum would be off
// by up to 2^-12 relative where one key dominates).
HN_DEVICE f32x16 step_a_lse(const f32x16& s, float c, float nm, float& l, f16x8 (&pf)[2], const uint8_t* ka,
                            const bf16x8 (&qf)[8]) {
    bf16x8 kf[8];
    kf[0] = ld_bf16x8(ka);
    kf[1] = ld_bf16x8(ka + 32);
    f32x16 acc;
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[v] = 0.0f;
    float ls = 0.0f;
    uint32_t x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (i + 2 < 8) kf[i + 2] = ld_bf16x8(ka + 32 * (i + 2));
        acc = mfma_bf16(kf[i], qf[i], acc);
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * i], c, nm));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * i + 1], c, nm));
        x[i] = pack_f16(p0, p1);
        ls += p0;
        ls += p1;
        pin(x[i], ls);
        __builtin_amdgcn_sched_barrier(0);
    }
    l += ls;
    pf[0] = __builtin_bit_cast(f16x8, make_uint4(x[0], x[1], x[2], x[3]));
    pf[1] = __builtin_bit_cast(f16x8, make_uint4(x[4], x[5], x[6], x[7]));
    return acc;
}

// The validity bits of this thread's quad keys, as 4 bits.
HN_DEVICE uint32_t quad_bits(uint64_t w) { return (uint32_t)(w >> quad_key(threadIdx.x & 15, 0)) & 15u; }

// V codes and scales of masked quad keys become zeros.
HN_DEVICE void clear_masked_v(CacheRegs<4>& r, float4& vs, uint64_t w) {
    const uint32_t m = quad_bits(w);
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (!((m >> j) & 1u)) r.v[j][0] = r.v[j][1] = 0u;
    vs.x = m & 1u ? vs.x : 0.0f;
    vs.y = m & 2u ? vs.y : 0.0f;
    vs.z = m & 4u ? vs.z : 0.0f;
    vs.w = m & 8u ? vs.w : 0.0f;
}

HN_DEVICE void clear_masked_v(TailRegs<4>& r, uint64_t w) {
    const uint32_t m = quad_bits(w);
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (!((m >> j) & 1u))
#pragma unroll
            for (int d = 0; d < 4; ++d) r.v[j][d] = 0u;
}

template <int FMT, bool MASK>
__global__ __launch_bounds__(256, 2) void attn_blocks_kernel(BlockParams p) {
    constexpr int NW = 4, BQ = Shape<NW>::BQ;
    __shared__ __attribute__((aligned(16))) uint8_t smem[smem_bytes<NW>()];
    float* const sbuf = reinterpret_cast<float*>(smem + 2 * STAGE);  // [2][128]

    // Work order as in attn_fp8kv_kernel: id % 8 (the XCD) picks a contiguous
    // range of items; without key splits the runs of a head are neighbours,
    // with them the heads of one key range.
    const int id = blockIdx.x;
    const int w = (id & 7) * p.per_xcd + (id >> 3);
    if (w >= p.work) return;
    int split, qt;
    int64_t h, b, run;
    if (p.splits > 1) {
        h = w % p.H;
        int x = w / (int)p.H;
        split = x % p.splits;
        x /= p.splits;
        qt = x % p.q_tiles;
        x /= p.q_tiles;
        run = x % p.runs;
        b = x / p.runs;
    } else {
        split = 0;
        qt = w % p.q_tiles;
        int x = w / p.q_tiles;
        run = x % p.runs;
        x /= (int)p.runs;
        h = x % p.H;
        b = x / p.H;
    }

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = lane & 31, half = lane >> 5;
    const int64_t i0 = run * p.q_block;
    const int64_t queries = p.Lq - i0 < p.q_block ? p.Lq - i0 : p.q_block;
    const int64_t rows = queries * p.G;  // of this run
    const int64_t row = (int64_t)qt * BQ + wave * QW + col;
    const bool qvalid = row < rows;
    const int64_t rr = qvalid ? row : rows - 1;
    const int64_t qi = i0 + rr / p.G, hq = h * p.G + rr % p.G;

    bf16x8 qf[8];
    {
        const uint16_t* src = p.q + b * p.qs0 + qi * p.qs1 + hq * p.qs2 + half * 8;
#pragma unroll
        for (int sl = 0; sl < 8; ++sl)
            qf[sl] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(src + 16 * sl));
    }

    const int32_t* list = p.idx ? p.idx + b * p.is0 + h * p.is1 + run * p.is2 : nullptr;
    const int n_cache = list ? list_length(list, p.top_k) << p.shift : (int)((p.kv_len + BKV - 1) / BKV);
    const int n_tail = (int)((p.cur_len + BKV - 1) / BKV);
    const int n_all = n_cache + n_tail;
    const int t_begin = (int)((int64_t)n_all * split / p.splits);
    const int t_end = (int)((int64_t)n_all * (split + 1) / p.splits);

    f32x16 o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[i][v] = 0.0f;
    Run run_{-INFINITY, 0.0f, 0.0f};
    const float c = p.scale_log2;

    // Tile t: segment, first key in it, keys that exist.
    struct Geom {
        bool cache;
        int64_t first;
        int count;
    };
    auto geom = [&](int t) {
        Geom g;
        int64_t left;
        if (t < n_cache) {
            g.cache = true;
            const int64_t e = list ? __builtin_amdgcn_readfirstlane(list[t >> p.shift]) : 0;
            g.first = list ? e * p.block + (int64_t)(t & ((1 << p.shift) - 1)) * BKV : (int64_t)t * BKV;
            left = p.kv_len - g.first;
        } else {
            g.cache = false;
            g.first = (int64_t)(t - n_cache) * BKV;
            left = p.cur_len - g.first;
        }
        g.count = left >= BKV ? BKV : left > 0 ? (int)left : 0;
        if (left <= 0) g.first = 0;  // an entry past the last block: nothing is read
        return g;
    };
    // The tile's keys that take part: existing and (MASK) valid.
    auto word_of = [&](const Geom& g, const uint8_t* st) {
        const uint64_t all = g.count >= BKV ? ALL_KEYS : (1ull << g.count) - 1;
        return tile_mask<MASK>(st) & all;
    };
    const uint32_t ka_off = col * KROW + 16 * half;
    const uint32_t va_off = K_BYTES + col * VTROW + 16 * half;
    CacheRegs<NW> regs;
    regs.s = 0.0f;
    const LaneOffs<NW> lo = lane_offsets<NW>(p);

    auto store_cache_tile = [&](const Geom& g, uint8_t* st, const float* sb) {  // prologue
        store_mask<NW, MASK>(regs, st);
        float ks[Shape<NW>::KU];
        k_scales<NW>(sb, ks);
        float4 vs = v_scales(sb);
        if constexpr (MASK) {
            __syncthreads();
            const uint64_t word = word_of(g, st);
            if (word != ALL_KEYS) clear_masked_v(regs, vs, word);
        }
        uint32_t kd[4];
        float vp[Shape<NW>::VD];
        uint32_t vd[2 * Shape<NW>::VD];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            store_k_part<FMT, NW>(regs, st, i, ks, kd);
            store_v_part<FMT, NW>(regs.v, st + K_BYTES, i, vs, vp, vd);
        }
    };
    auto copy_tail = [&](const Geom& g, uint8_t* st) {  // prologue and the first tail tile
        TailRegs<NW> r;
        load_tail_k<NW, MASK>(p, b, h, g.first, g.count, r);
        load_tail_v<NW>(p, b, h, g.first, g.count, r);
        store_tail_k<NW, MASK>(r, st);
        if constexpr (MASK) {
            __syncthreads();
            const uint64_t word = word_of(g, st);
            if (word != ALL_KEYS) clear_masked_v(r, word);
        }
        store_tail_v<NW>(r, st);
    };

    if (t_end > t_begin) {
        f32x16 sa, sb;
        float mxa, mxb;
        uint64_t mw;
        Geom g = geom(t_begin);
        if (g.cache) {
            const TileBase tb = tile_base(p, b, h, g.first, g.count);
            load_k<NW, MASK>(lo, regs, tb, g.count);
            load_v<NW>(lo, regs, tb);
            __builtin_amdgcn_s_waitcnt(0);
            if (threadIdx.x < 2 * BKV) sbuf[threadIdx.x] = regs.s;
            __syncthreads();
            store_cache_tile(g, smem, sbuf);
        } else {
            copy_tail(g, smem);
        }
        Geom gn = geom(t_begin + 1 < t_end ? t_begin + 1 : t_begin);
        if (t_begin + 1 < t_end && gn.cache) {
            const TileBase tb = tile_base(p, b, h, gn.first, gn.count);
            load_k<NW, MASK>(lo, regs, tb, gn.count);
            load_v<NW>(lo, regs, tb);
        }
        __builtin_amdgcn_s_waitcnt(0);
        if (threadIdx.x < 2 * BKV) sbuf[SB_FLOATS + threadIdx.x] = regs.s;
        __syncthreads();
        mw = word_of(g, smem);
        sa = s_block(smem + ka_off, qf);
        mxa = raw_max(sa);
        if ((uint32_t)mw != ~0u) mxa = mask_word(sa, (uint32_t)mw);
        int t = t_begin;
        // Cache tiles, and the step into the tail.
        for (; t < t_end && t < n_cache; ++t) {
            const int u = t - t_begin;
            const uint8_t* st = smem + (u & 1) * STAGE;
            uint8_t* nst = smem + ((u & 1) ^ 1) * STAGE;
            const float* nsb = sbuf + ((u & 1) ^ 1) * SB_FLOATS;
            const bool has_next = t + 1 < t_end;
            const Geom g2 = geom(t + 2 < t_end ? t + 2 : t_end - 1);
            const int n2 = t + 2 < t_end && g2.cache ? g2.count : 0;  // 0: no fetch (zeros)
            f16x8 pf[2];
            // ---- half 0
            rebase(mxa, c, run_, o);
            sb = step_a_lse(sa, c, run_.nm, run_.l, pf, st + ka_off + 32 * KROW, qf);
            {
                float ks[Shape<NW>::KU];
                k_scales<NW>(nsb, ks);
                uint32_t kd[4];
                mxb = step_b_with(pf, st + va_off, 0, o, sb, [&](int i) __attribute__((always_inline)) {
                    store_k_part<FMT, NW>(regs, nst, i, ks, kd);
                });
            }
            store_mask<NW, MASK>(regs, nst);
            if ((uint32_t)(mw >> 32) != ~0u) mxb = mask_word(sb, (uint32_t)(mw >> 32));
            const bool tail_next = has_next && !gn.cache;
            TailRegs<NW> tr;
            if (tail_next) {
                load_tail_k<NW, MASK>(p, b, h, gn.first, gn.count, tr);
                store_tail_k<NW, MASK>(tr, nst);
            }
            const TileBase tb2 = tile_base(p, b, h, g2.first, n2);
            load_k<NW, MASK>(lo, regs, tb2, n2);
            __syncthreads();
            // ---- half 1 (on the last tile the S block of "tile t + 1" reads stale
            // LDS; its result is never used)
            const uint64_t mwn = word_of(gn, nst);
            rebase(mxb, c, run_, o);
            sa = step_a_lse(sb, c, run_.nm, run_.l, pf, nst + ka_off, qf);
            {
                float4 vs = v_scales(nsb);
                if constexpr (MASK)
                    if (mwn != ALL_KEYS) clear_masked_v(regs, vs, mwn);
                float vp[Shape<NW>::VD];
                uint32_t vd[2 * Shape<NW>::VD];
                mxa = step_b_with(pf, st + va_off, 1, o, sa, [&](int i) __attribute__((always_inline)) {
                    store_v_part<FMT, NW>(regs.v, nst + K_BYTES, i, vs, vp, vd);
                });
            }
            if ((uint32_t)mwn != ~0u) mxa = mask_word(sa, (uint32_t)mwn);
            if (tail_next) {
                load_tail_v<NW>(p, b, h, gn.first, gn.count, tr);
                if constexpr (MASK)
                    if (mwn != ALL_KEYS) clear_masked_v(tr, mwn);
                store_tail_v<NW>(tr, nst);
            }
            if (threadIdx.x < 2 * BKV) sbuf[(u & 1) * SB_FLOATS + threadIdx.x] = regs.s;
            load_v<NW>(lo, regs, tb2);
            __syncthreads();
            g = gn;
            gn = g2;
            mw = mwn;
        }
        // Tail tiles.
        if (t < t_end) {
            TailRegs<NW> tr;
            auto fetch_k = [&](int tt) {
                if (tt < t_end) load_tail_k<NW, MASK>(p, b, h, (int64_t)(tt - n_cache) * BKV, geom(tt).count, tr);
            };
            auto fetch_v = [&](int tt) {
                if (tt < t_end) load_tail_v<NW>(p, b, h, (int64_t)(tt - n_cache) * BKV, geom(tt).count, tr);
            };
            fetch_k(t + 1);
            fetch_v(t + 1);
            for (; t < t_end; ++t) {
                const int u = t - t_begin;
                const uint8_t* st = smem + (u & 1) * STAGE;
                uint8_t* nst = smem + ((u & 1) ^ 1) * STAGE;
                const bool has_next = t + 1 < t_end;
                f16x8 pf[2];
                rebase(mxa, c, run_, o);
                sb = step_a_lse(sa, c, run_.nm, run_.l, pf, st + ka_off + 32 * KROW, qf);
                mxb = step_b_with(pf, st + va_off, 0, o, sb, [&](int i) __attribute__((always_inline)) {
                    if ((i & 1) && has_next) store_tail_k_part<NW>(tr, nst, i >> 2, (i >> 1) & 1);
                });
                if (has_next) store_tail_mask<NW, MASK>(tr, nst);
                if ((uint32_t)(mw >> 32) != ~0u) mxb = mask_word(sb, (uint32_t)(mw >> 32));
                fetch_k(t + 2);
                __syncthreads();
                const uint64_t mwn = word_of(geom(has_next ? t + 1 : t), nst);
                if constexpr (MASK)
                    if (mwn != ALL_KEYS && has_next) clear_masked_v(tr, mwn);
                rebase(mxb, c, run_, o);
                sa = step_a_lse(sb, c, run_.nm, run_.l, pf, nst + ka_off, qf);
                mxa = step_b_with(pf, st + va_off, 1, o, sa, [&](int i) __attribute__((always_inline)) {
                    if (has_next) store_tail_v_part<NW>(tr, nst, i);
                });
                if ((uint32_t)mwn != ~0u) mxa = mask_word(sa, (uint32_t)mwn);
                fetch_v(t + 2);
                __syncthreads();
                mw = mwn;
            }
        }
    }
    const float l = run_.l + __shfl_xor(run_.l, 32, 64);
    const float m = run_.m;
    if (!qvalid) return;
    const int64_t hqs = p.H * p.G, at = (b * hqs + hq) * p.Lq + qi;
    if (p.splits > 1) {
        const int64_t slot = (int64_t)split * p.B * hqs * p.Lq + at;
        float* dst = p.ws_o + slot * D;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int vq = 0; vq < 4; ++vq)
                *reinterpret_cast<float4*>(dst + db * 32 + vq * 8 + half * 4) =
                    make_float4(o[db][vq * 4], o[db][vq * 4 + 1], o[db][vq * 4 + 2], o[db][vq * 4 + 3]);
        if (half == 0) *reinterpret_cast<float2*>(p.ws_ml + slot * 2) = make_float2(m, l);
        return;
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    uint16_t* dst = p.out + b * p.os0 + qi * p.os1 + hq * p.os2;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int vq = 0; vq < 4; ++vq) {
            const int d = db * 32 + vq * 8 + half * 4;
            *reinterpret_cast<uint2*>(dst + d) =
                make_uint2(pack_bf16(o[db][vq * 4] * inv, o[db][vq * 4 + 1] * inv),
                           pack_bf16(o[db][vq * 4 + 2] * inv, o[db][vq * 4 + 3] * inv));
        }
    if (half == 0) p.lse[at] = l > 0.0f ? (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f : -INFINITY;
}

// Merge of the key splits (as attn_combine_kernel), with the row's log-sum-exp.
__global__ __launch_bounds__(256) void blocks_combine_kernel(BlockParams p) {
    const int64_t hqs = p.H * p.G, rows = p.B * hqs * p.Lq;
    const int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);  // (b * Hq + hq) * Lq + i
    if (r >= rows) return;
    const int d = (threadIdx.x & 31) * 4;
    float M = -INFINITY;
    for (int sp = 0; sp < p.splits; ++sp) M = fmaxf(M, p.ws_ml[(sp * rows + r) * 2]);
    const float base = M == -INFINITY ? 0.0f : M;
    float den = 0.0f, num[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int sp = 0; sp < p.splits; ++sp) {
        const int64_t at = sp * rows + r;
        const float2 ml = *reinterpret_cast<const float2*>(p.ws_ml + at * 2);
        const float4 ov = *reinterpret_cast<const float4*>(p.ws_o + at * D + d);
        const float wgt = __builtin_amdgcn_exp2f(ml.x - base);
        den = fmaf(wgt, ml.y, den);
        num[0] = fmaf(wgt, ov.x, num[0]);
        num[1] = fmaf(wgt, ov.y, num[1]);
        num[2] = fmaf(wgt, ov.z, num[2]);
        num[3] = fmaf(wgt, ov.w, num[3]);
    }
    const int64_t i = r % p.Lq, hq = (r / p.Lq) % hqs, b = r / (p.Lq * hqs);
    const float inv = den > 0.0f ? 1.0f / den : 0.0f;
    *reinterpret_cast<uint2*>(p.out + b * p.os0 + i * p.os1 + hq * p.os2 + d) =
        make_uint2(pack_bf16(num[0] * inv, num[1] * inv), pack_bf16(num[2] * inv, num[3] * inv));
    if (d == 0) p.lse[r] = den > 0.0f ? (base + __builtin_amdgcn_logf(den)) * 0.6931471805599453f : -INFINITY;
}

// ---------------------------------------------------------------------------
// Key mass. A wave holds 32 KB keys as MFMA operands in registers; the query rows
// stream past them through LDS, 32 at a time. S = Q K^T puts one key per lane
// column, so a key's mass is a sum over the lane's own registers and one exchange
// with lane ^ 32 at the end; the rows' log-sum-exps come as four 16-byte LDS reads
// a tile. The MFMAs of one key block run beside the exponentials of the one before.
// One workgroup sees every row of its keys (or, split, its share of the rows, added
// in order afterwards), so no two add to one key and the result has one order.
struct MassParams {
    const uint16_t* q;
    const float* lse;       // [Bq, Hq, Lq]
    const uint8_t* kc;
    const float* ks;
    const uint8_t* valid;
    const float* prior;     // [B, H, prior_len] or null
    float* mass;            // [B, H, kv_len]
    int64_t qs0, qs1, qs2, cs0, cs1, cs2, ss0, ss1, ss2, vs, ps0, ps1;
    int64_t Lq, kv_len, prior_len;
    int64_t rows;           // query rows per cached head: batches * Lq * G
    int64_t rows_per_split; // rows of a workgroup (a multiple of MASS_ROWS)
    float* part;            // row splits: [split][B, H, kv_len] sums, or null
    int64_t B;
    int batches;            // query batches per cache slot
    int H, G, tiles, work, per_xcd;
    float scale_log2;
};

constexpr int MASS_ROWS = 32;   // query rows per LDS tile
constexpr int MASS_TILE = MASS_ROWS * KROW;

// The exponentials of block s (rows' n = -lse log2 e) beside the S of the next block.
HN_DEVICE f32x16 mass_step(const f32x16& s, float c, const f32x16& n, float& acc, const bf16x8 (&qf)[8],
                           const bf16x8 (&kf)[8]) {
    f32x16 next;
#pragma unroll
    for (int v = 0; v < 16; ++v) next[v] = 0.0f;
    float a0 = 0.0f, a1 = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        next = mfma_bf16(qf[i], kf[i], next);
        a0 += __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * i], c, n[2 * i]));
        a1 += __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * i + 1], c, n[2 * i + 1]));
        pin(a0, a1);
        __builtin_amdgcn_sched_barrier(0);
    }
    acc += a0 + a1;
    return next;
}

template <int FMT, int KB>
__global__ __launch_bounds__(256, 2) void key_mass_kernel(MassParams p) {
    __shared__ __attribute__((aligned(16))) uint8_t smem[2 * MASS_TILE];
    __shared__ __attribute__((aligned(16))) float nl[2][MASS_ROWS];
    // Work order: id % 8 (the XCD) picks a contiguous range of items, heads fastest:
    // the heads of one key range share the lines of its scales in one L2.
    const int w = (int)(blockIdx.x & 7) * p.per_xcd + (int)(blockIdx.x >> 3);
    if (w >= p.work) return;
    const int64_t h = w % p.H;
    int x = w / p.H;
    const int tile = x % p.tiles;
    x /= p.tiles;
    const int64_t b = x % p.B, split = x / p.B;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, half = lane >> 5;
    const int64_t key0 = ((int64_t)tile * 4 + wave) * (32 * KB);
    const float c = p.scale_log2;

    // K fragments: key 32 kb + col, dims 64 half + 8 sl ..: 64 contiguous bytes a lane
    bf16x8 kf[KB][8];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
        const int64_t key = key0 + 32 * kb + col;
        uint4 y[4];
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = make_uint4(0u, 0u, 0u, 0u);
        if (key < p.kv_len && (!p.valid || p.valid[b * p.vs + key] != 0)) {
            const uint4* src = reinterpret_cast<const uint4*>(p.kc + b * p.cs0 + key * p.cs1 + h * p.cs2 + 64 * half);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = src[e];
            s = p.ks[b * p.ss0 + key * p.ss1 + h * p.ss2];
        }
#pragma unroll
        for (int sl = 0; sl < 8; ++sl) {
            uint32_t d[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const f32x2 f = codes2_f32<FMT>(word(y[sl >> 1], 2 * (sl & 1) + (e >> 1)), e & 1);
                d[e] = pack_bf16(f[0] * s, f[1] * s);
            }
            kf[kb][sl] = __builtin_bit_cast(bf16x8, make_uint4(d[0], d[1], d[2], d[3]));
        }
    }

    // This thread's 32 bytes of a query tile: row tid / 8, dims 16 (tid % 8) ..
    const int tr = tid >> 3, tu = tid & 7;
    const int64_t row0 = split * p.rows_per_split;
    const int64_t row1 = row0 + p.rows_per_split < p.rows ? row0 + p.rows_per_split : p.rows;
    uint4 x0, x1;
    float ln = 0.0f;
    // Row r0 + tr of the next fetch: query head g of the group, query i, batch bb; each
    // fetch moves 32 rows on (steps dg, di, db with their carries; no division).
    int64_t r = row0 + tr;
    int g = (int)(r % p.G);
    int64_t i = p.Lq > 0 ? (r / p.G) % p.Lq : 0, bb = b * p.batches + (p.Lq > 0 ? r / (p.G * p.Lq) : 0);
    const int dg = MASS_ROWS % p.G;
    const int64_t di = p.Lq > 0 ? (MASS_ROWS / p.G) % p.Lq : 0, db = p.Lq > 0 ? MASS_ROWS / p.G / p.Lq : 0;
    auto fetch = [&]() {
        x0 = x1 = make_uint4(0u, 0u, 0u, 0u);
        ln = -INFINITY;  // a row that adds nothing: exp2(0 - inf) = 0
        if (r < row1) {
            const float lse = p.lse[(bb * p.H * p.G + h * p.G + g) * p.Lq + i];
            if (__builtin_fabsf(lse) != INFINITY) {
                ln = -lse * 1.4426950408889634f;
                const uint16_t* src = p.q + bb * p.qs0 + i * p.qs1 + (h * p.G + g) * p.qs2 + 16 * tu;
                x0 = reinterpret_cast<const uint4*>(src)[0];
                x1 = reinterpret_cast<const uint4*>(src)[1];
            }
        }
        r += MASS_ROWS;
        g += dg;
        i += di;
        bb += db;
        if (g >= p.G) {
            g -= p.G;
            ++i;
        }
        if (i >= p.Lq) {
            i -= p.Lq;
            ++bb;
        }
    };
    auto put = [&](int buf) {
        uint4* dst = reinterpret_cast<uint4*>(smem + buf * MASS_TILE + tr * KROW + 32 * tu);
        dst[0] = x0;
        dst[1] = x1;
        if (tu == 0) nl[buf][tr] = ln;
    };
    float acc[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) acc[kb] = 0.0f;
    fetch();
    put(0);
    __syncthreads();
    int buf = 0;
    for (int64_t r0 = row0; r0 < row1; r0 += MASS_ROWS, buf ^= 1) {
        const bool more = r0 + MASS_ROWS < row1;
        if (more) fetch();
        bf16x8 qf[8];
        const uint8_t* qa = smem + buf * MASS_TILE + col * KROW + 128 * half;
#pragma unroll
        for (int sl = 0; sl < 8; ++sl) qf[sl] = ld_bf16x8(qa + 16 * sl);
        f32x16 n;  // row 8 (v / 4) + 4 half + v % 4
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float4 y = *reinterpret_cast<const float4*>(&nl[buf][8 * e + 4 * half]);
            n[4 * e] = y.x;
            n[4 * e + 1] = y.y;
            n[4 * e + 2] = y.z;
            n[4 * e + 3] = y.w;
        }
        f32x16 s;
#pragma unroll
        for (int v = 0; v < 16; ++v) s[v] = 0.0f;
#pragma unroll
        for (int sl = 0; sl < 8; ++sl) s = mfma_bf16(qf[sl], kf[0][sl], s);
#pragma unroll
        for (int kb = 1; kb < KB; ++kb) s = mass_step(s, c, n, acc[kb - 1], qf, kf[kb]);
        float a0 = 0.0f, a1 = 0.0f;
#pragma unroll
        for (int v = 0; v < 16; v += 2) {
            a0 += __builtin_amdgcn_exp2f(__builtin_fmaf(s[v], c, n[v]));
            a1 += __builtin_amdgcn_exp2f(__builtin_fmaf(s[v + 1], c, n[v + 1]));
        }
        acc[KB - 1] += a0 + a1;
        if (more) put(buf ^ 1);
        __syncthreads();
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
        const float s = acc[kb] + __shfl_xor(acc[kb], 32, 64);
        const int64_t key = key0 + 32 * kb + col;
        if (half != 0 || key >= p.kv_len) continue;
        if (p.part) {
            p.part[((split * p.B + b) * p.H + h) * p.kv_len + key] = s;
            continue;
        }
        const bool ok = !p.valid || p.valid[b * p.vs + key] != 0;
        const float before = p.prior && key < p.prior_len ? p.prior[b * p.ps0 + h * p.ps1 + key] : 0.0f;
        p.mass[(b * p.H + h) * p.kv_len + key] = ok ? before + s : before;
    }
}

// Sum of the row splits in order, onto the prior mass.
__global__ __launch_bounds__(256) void key_mass_sum_kernel(MassParams p, int splits) {
    const int64_t key = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (key >= p.kv_len) return;
    const int64_t h = blockIdx.y % p.H, b = blockIdx.y / p.H;
    float s = 0.0f;
    for (int sp = 0; sp < splits; ++sp) s += p.part[((int64_t)sp * gridDim.y + blockIdx.y) * p.kv_len + key];
    const bool ok = !p.valid || p.valid[b * p.vs + key] != 0;
    const float before = p.prior && key < p.prior_len ? p.prior[b * p.ps0 + h * p.ps1 + key] : 0.0f;
    p.mass[(int64_t)blockIdx.y * p.kv_len + key] = ok ? before + s : before;
}

}  // namespace attn
}  // namespace hn

using namespace hn;

// Key splits: a launch wants two workgroups per CU (two fit by LDS and
// registers); where the runs fall short, each workgroup's tiles are split.
// Each split keeps at least 4 tiles: a split of fewer costs more in its prologue
// and in the merge than the wider grid gives.
static int blocks_splits(int64_t work, int64_t tiles) {
    const int64_t target = 2LL * device_cus();
    if (work <= 0 || work >= target) return 1;
    int64_t sp = target / work;
    if (sp > tiles / 4) sp = tiles / 4;
    return sp > 1 ? (int)sp : 1;
}

struct BlocksPlan {
    int64_t runs, q_tiles, work;
    int splits;
};

static BlocksPlan blocks_plan(int64_t B, int64_t Lq, int64_t Hq, int64_t H, int64_t kv_len, int64_t cur_len,
                              int64_t top_k, int64_t block, int64_t q_block) {
    BlocksPlan pl;
    pl.runs = (Lq - 1) / q_block + 1;
    const int64_t rows = (q_block < Lq ? q_block : Lq) * (Hq / H);
    pl.q_tiles = (rows + attn::Shape<4>::BQ - 1) / attn::Shape<4>::BQ;
    pl.work = B * H * pl.runs * pl.q_tiles;
    const int64_t listed = top_k >= 0 ? top_k * (block / attn::BKV) : (kv_len + attn::BKV - 1) / attn::BKV;
    pl.splits = blocks_splits(pl.work, listed + (cur_len + attn::BKV - 1) / attn::BKV);
    return pl;
}

static bool blocks_shape_ok(int64_t B, int64_t Lq, int64_t Hq, int64_t H, int64_t kv_len, int64_t cur_len,
                            int64_t block, int64_t q_block) {
    return B > 0 && Lq > 0 && H > 0 && Hq > 0 && Hq % H == 0 && kv_len >= 0 && cur_len >= 0 && block >= 64 &&
           block <= 1024 && (block & (block - 1)) == 0 && q_block > 0;
}

extern "C" int64_t hn_attn_kv_blocks_workspace_size(int64_t B, int64_t Lq, int64_t Hq, int64_t H, int64_t kv_len,
                                                    int64_t cur_len, int64_t top_k, int64_t block, int64_t q_block) {
    if (!blocks_shape_ok(B, Lq, Hq, H, kv_len, cur_len, block, q_block)) return 0;
    const BlocksPlan pl = blocks_plan(B, Lq, Hq, H, kv_len, cur_len, top_k, block, q_block);
    return pl.splits > 1 ? (int64_t)pl.splits * B * Hq * Lq * (attn::D + 2) * (int64_t)sizeof(float) : 0;
}

extern "C" int hn_attn_kv_blocks(int fmt, const void* q, const int64_t* qs, int64_t B, int64_t Lq, int64_t Hq,
                                 int64_t D, const void* kc, const void* vc, const int64_t* cs, const float* ks,
                                 const float* vs, const int64_t* ss, int64_t H, int64_t cache_cap, int64_t kv_len,
                                 const uint8_t* cache_valid, int64_t cache_valid_stride, const int32_t* idx,
                                 const int64_t* is, int64_t top_k, int64_t block, int64_t q_block, const void* kcur,
                                 const void* vcur, const int64_t* curs, int64_t cur_len, const uint8_t* cur_valid,
                                 int64_t cur_valid_stride, float softmax_scale, void* out, const int64_t* os,
                                 float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
    HN_REQUIRE(fmt == HN_KV_FP8 || fmt == HN_KV_INT8, HN_E_ARG, "hn_attn_kv_blocks: unknown KV format");
    HN_REQUIRE(D == attn::D, HN_E_ARG, "hn_attn_kv_blocks: head dim must be 128");
    HN_REQUIRE(B >= 0 && Lq >= 0 && H > 0 && Hq > 0 && Hq % H == 0 && kv_len >= 0 && cur_len >= 0, HN_E_ARG,
               "hn_attn_kv_blocks: invalid shape");
    HN_REQUIRE(block >= 64 && block <= 1024 && (block & (block - 1)) == 0, HN_E_ARG,
               "hn_attn_kv_blocks: block must be 64, 128, 256, 512 or 1024");
    HN_REQUIRE(q_block > 0, HN_E_ARG, "hn_attn_kv_blocks: q_block must be positive");
    HN_REQUIRE(kv_len <= cache_cap, HN_E_ARG, "hn_attn_kv_blocks: kv_len exceeds the cache capacity");
    HN_REQUIRE(kv_len <= 0x3fffffffLL && cur_len <= 0x3fffffffLL && (!idx || (top_k >= 0 && top_k <= 0x3fffffLL)),
               HN_E_ARG, "hn_attn_kv_blocks: too many keys");
    HN_REQUIRE(softmax_scale > 0.0f && softmax_scale <= 3.4028234e38f, HN_E_ARG,
               "hn_attn_kv_blocks: softmax_scale must be finite and positive");
    HN_REQUIRE(cache_valid_stride >= 0 && cur_valid_stride >= 0, HN_E_ARG, "hn_attn_kv_blocks: negative validity stride");
    HN_REQUIRE(qs && os && (kv_len == 0 || (cs && ss)) && (cur_len == 0 || curs) && (!idx || is), HN_E_ARG,
               "hn_attn_kv_blocks: null stride array");
    HN_REQUIRE(qs[3] == 1 && os[3] == 1, HN_E_ARG, "hn_attn_kv_blocks: head dim must be contiguous");
    HN_REQUIRE(qs[0] % 8 == 0 && qs[1] % 8 == 0 && qs[2] % 8 == 0 && os[0] % 4 == 0 && os[1] % 4 == 0 && os[2] % 4 == 0,
               HN_E_ARG, "hn_attn_kv_blocks: q/out strides misaligned");
    HN_REQUIRE(aligned(q, 16) && aligned(out, 8) && aligned(idx, 4) && aligned(lse, 4), HN_E_ARG,
               "hn_attn_kv_blocks: q/out misaligned");
    if (kv_len > 0) {
        HN_REQUIRE(kc && vc && ks && vs, HN_E_ARG, "hn_attn_kv_blocks: null cache pointer");
        HN_REQUIRE(cs[3] == 1 && cs[0] % 16 == 0 && cs[1] % 16 == 0 && cs[2] % 16 == 0, HN_E_ARG,
                   "hn_attn_kv_blocks: cache strides must be multiples of 16 bytes");
        HN_REQUIRE(cs[0] >= 0 && cs[1] > 0 && cs[2] >= 0 && ss[0] >= 0 && ss[1] > 0 && ss[2] >= 0 &&
                       cs[1] <= 0x1ffffffLL && ss[1] <= 0x7fffffLL,
                   HN_E_ARG, "hn_attn_kv_blocks: invalid cache strides");
        HN_REQUIRE(aligned(kc, 16) && aligned(vc, 16), HN_E_ARG, "hn_attn_kv_blocks: cache misaligned");
    }
    if (cur_len > 0) {
        HN_REQUIRE(kcur && vcur, HN_E_ARG, "hn_attn_kv_blocks: null tail pointer");
        HN_REQUIRE(curs[3] == 1 && curs[0] % 8 == 0 && curs[1] % 8 == 0 && curs[2] % 8 == 0, HN_E_ARG,
                   "hn_attn_kv_blocks: tail strides must be multiples of 8");
        HN_REQUIRE(aligned(kcur, 16) && aligned(vcur, 16), HN_E_ARG, "hn_attn_kv_blocks: tail misaligned");
    }
    if (B == 0 || Lq == 0) return HN_OK;
    HN_REQUIRE(q && out && lse, HN_E_ARG, "hn_attn_kv_blocks: null q/out/lse");
    const BlocksPlan pl = blocks_plan(B, Lq, Hq, H, kv_len, cur_len, idx ? top_k : -1, block, q_block);
    const int64_t need = pl.splits > 1 ? (int64_t)pl.splits * B * Hq * Lq * (attn::D + 2) * (int64_t)sizeof(float) : 0;
    HN_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned(workspace, 16))), HN_E_ARG,
               "hn_attn_kv_blocks: workspace smaller than hn_attn_kv_blocks_workspace_size() or misaligned");
    const int64_t work = pl.work * pl.splits;
    HN_REQUIRE(work <= 0x3fffffffLL && pl.runs <= 0x3fffffffLL && B * Hq * Lq <= 0x3ffffffffLL, HN_E_ARG,
               "hn_attn_kv_blocks: too much work for one launch");
    if (const int rc = require_gfx950("hn_attn_kv_blocks"); rc != HN_OK) return rc;
    attn::BlockParams p = {};
    p.q = (const uint16_t*)q; p.out = (uint16_t*)out; p.lse = lse;
    p.kc = (const uint8_t*)kc; p.vc = (const uint8_t*)vc; p.ks = ks; p.vs = vs;
    p.kcur = (const uint16_t*)kcur; p.vcur = (const uint16_t*)vcur;
    p.kvalid = kv_len > 0 ? cache_valid : nullptr;
    p.uvalid = cur_len > 0 ? cur_valid : nullptr;
    p.kvs = cache_valid_stride; p.uvs = cur_valid_stride;
    p.qs0 = qs[0]; p.qs1 = qs[1]; p.qs2 = qs[2];
    p.os0 = os[0]; p.os1 = os[1]; p.os2 = os[2];
    if (kv_len > 0) {
        p.cs0 = cs[0]; p.cs1 = cs[1]; p.cs2 = cs[2];
        p.ss0 = ss[0]; p.ss1 = ss[1]; p.ss2 = ss[2];
    }
    if (cur_len > 0) {
        p.us0 = curs[0]; p.us1 = curs[1]; p.us2 = curs[2];
    }
    p.Lq = Lq; p.H = H; p.G = (int)(Hq / H); p.B = B; p.kv_len = kv_len; p.cur_len = cur_len;
    p.scale_log2 = softmax_scale * 1.4426950408889634f;
    p.fmt = fmt;
    p.idx = kv_len > 0 ? idx : nullptr;
    if (idx && kv_len > 0) {
        p.is0 = is[0]; p.is1 = is[1]; p.is2 = is[2];
    }
    p.top_k = (int)(idx ? top_k : 0);
    p.block = block;
    p.shift = __builtin_ctzll((unsigned long long)block) - 6;
    p.q_block = q_block; p.runs = pl.runs;
    p.q_tiles = (int)pl.q_tiles; p.splits = pl.splits;
    p.work = (int)work;
    p.per_xcd = (int)((work + 7) / 8);
    if (pl.splits > 1) {
        p.ws_o = (float*)workspace;
        p.ws_ml = (float*)workspace + (int64_t)pl.splits * B * Hq * Lq * attn::D;
    }
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)(8 * (int64_t)p.per_xcd));
    const bool mask = p.kvalid || p.uvalid;
    if (fmt == HN_KV_FP8) {
        if (mask) attn::attn_blocks_kernel<HN_KV_FP8, true><<<grid, 256, 0, st>>>(p);
        else attn::attn_blocks_kernel<HN_KV_FP8, false><<<grid, 256, 0, st>>>(p);
    } else {
        if (mask) attn::attn_blocks_kernel<HN_KV_INT8, true><<<grid, 256, 0, st>>>(p);
        else attn::attn_blocks_kernel<HN_KV_INT8, false><<<grid, 256, 0, st>>>(p);
    }
    const int rc = check_launch("hn_attn_kv_blocks");
    if (rc != HN_OK || pl.splits == 1) return rc;
    attn::blocks_combine_kernel<<<(unsigned)((B * Hq * Lq + 7) / 8), 256, 0, st>>>(p);
    return check_launch("hn_attn_kv_blocks (combine)");
}

// Plan of the key mass: 512 keys per workgroup (KB 4), or 128 (KB 1) where those
// would not fill the device twice over; where even these fall short (a short cache,
// many queries) the rows are split, each split writes its sums and a second kernel
// adds them in order.
struct MassPlan {
    int kb, splits;
    int64_t tiles;
};

static MassPlan mass_plan(int64_t rows, int64_t B, int64_t H, int64_t kv_len) {
    const int64_t target = 2LL * device_cus();
    MassPlan pl{4, 1, (kv_len + 511) / 512};
    if (B * H * pl.tiles >= target) return pl;
    pl.kb = 1;
    pl.tiles = (kv_len + 127) / 128;
    const int64_t work = B * H * pl.tiles;
    int64_t sp = work > 0 ? target / work : 1;
    const int64_t cap = rows / (4 * attn::MASS_ROWS);  // at least 4 row tiles each
    if (sp > cap) sp = cap;
    pl.splits = sp > 1 ? (int)sp : 1;
    return pl;
}

extern "C" int64_t hn_attn_key_mass_workspace_size(int64_t Bq, int64_t Lq, int64_t Hq, int64_t B, int64_t H,
                                                   int64_t kv_len) {
    if (Bq <= 0 || Lq <= 0 || B <= 0 || H <= 0 || Hq <= 0 || Hq % H != 0 || Bq % B != 0 || kv_len <= 0) return 0;
    const int sp = mass_plan(Bq / B * Lq * (Hq / H), B, H, kv_len).splits;
    return sp > 1 ? (int64_t)sp * B * H * kv_len * (int64_t)sizeof(float) : 0;
}

extern "C" int hn_attn_key_mass(int fmt, const void* q, const int64_t* qs, int64_t Bq, int64_t Lq, int64_t Hq,
                                int64_t D, const float* lse, const void* kc, const int64_t* cs, const float* ks,
                                const int64_t* ss, int64_t B, int64_t H, int64_t cache_cap, int64_t kv_len,
                                const uint8_t* cache_valid, int64_t cache_valid_stride, float softmax_scale,
                                const float* prior, const int64_t* ps, int64_t prior_len, float* mass,
                                void* workspace, int64_t workspace_bytes, void* stream) {
    HN_REQUIRE(fmt == HN_KV_FP8 || fmt == HN_KV_INT8, HN_E_ARG, "hn_attn_key_mass: unknown KV format");
    HN_REQUIRE(D == attn::D, HN_E_ARG, "hn_attn_key_mass: head dim must be 128");
    HN_REQUIRE(B >= 0 && Bq >= 0 && Lq >= 0 && H > 0 && Hq > 0 && Hq % H == 0 && kv_len >= 0 && prior_len >= 0, HN_E_ARG,
               "hn_attn_key_mass: invalid shape");
    HN_REQUIRE(B == 0 || Bq % B == 0, HN_E_ARG, "hn_attn_key_mass: query batches do not divide into the cache's");
    HN_REQUIRE(kv_len <= cache_cap && kv_len <= 0x3fffffffLL, HN_E_ARG, "hn_attn_key_mass: kv_len exceeds the cache capacity");
    HN_REQUIRE(prior_len <= kv_len, HN_E_ARG, "hn_attn_key_mass: the prior mass is longer than the cache");
    HN_REQUIRE(softmax_scale > 0.0f && softmax_scale <= 3.4028234e38f, HN_E_ARG,
               "hn_attn_key_mass: softmax_scale must be finite and positive");
    HN_REQUIRE(cache_valid_stride >= 0, HN_E_ARG, "hn_attn_key_mass: negative validity stride");
    HN_REQUIRE(qs && cs && ss && (prior_len == 0 || ps), HN_E_ARG, "hn_attn_key_mass: null stride array");
    HN_REQUIRE(qs[3] == 1 && qs[0] % 8 == 0 && qs[1] % 8 == 0 && qs[2] % 8 == 0, HN_E_ARG,
               "hn_attn_key_mass: q strides misaligned");
    HN_REQUIRE(cs[3] == 1 && cs[0] % 16 == 0 && cs[1] % 16 == 0 && cs[2] % 16 == 0, HN_E_ARG,
               "hn_attn_key_mass: cache strides must be multiples of 16 bytes");
    HN_REQUIRE(aligned(q, 16) && aligned(kc, 16), HN_E_ARG, "hn_attn_key_mass: misaligned pointer");
    if (B == 0 || kv_len == 0) return HN_OK;
    HN_REQUIRE(kc && ks && mass && (prior_len == 0 || prior) && (Bq * Lq == 0 || (q && lse)), HN_E_ARG,
               "hn_attn_key_mass: null pointer");
    const int64_t need = hn_attn_key_mass_workspace_size(Bq, Lq, Hq, B, H, kv_len);
    HN_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned(workspace, 16))), HN_E_ARG,
               "hn_attn_key_mass: workspace smaller than hn_attn_key_mass_workspace_size() or misaligned");
    HN_REQUIRE(B * H <= 65535, HN_E_ARG, "hn_attn_key_mass: too many heads for one launch");
    if (const int rc = require_gfx950("hn_attn_key_mass"); rc != HN_OK) return rc;
    attn::MassParams p = {};
    p.q = (const uint16_t*)q; p.lse = lse; p.kc = (const uint8_t*)kc; p.ks = ks;
    p.valid = cache_valid; p.prior = prior_len ? prior : nullptr; p.mass = mass;
    p.qs0 = qs[0]; p.qs1 = qs[1]; p.qs2 = qs[2];
    p.cs0 = cs[0]; p.cs1 = cs[1]; p.cs2 = cs[2];
    p.ss0 = ss[0]; p.ss1 = ss[1]; p.ss2 = ss[2];
    p.vs = cache_valid_stride;
    if (prior_len) {
        p.ps0 = ps[0]; p.ps1 = ps[1];
    }
    p.Lq = Lq; p.kv_len = kv_len; p.prior_len = prior_len;
    p.batches = (int)(Bq / B);
    p.H = (int)H; p.G = (int)(Hq / H);
    p.rows = (int64_t)p.batches * Lq * p.G;
    p.scale_log2 = softmax_scale * 1.4426950408889634f;
    const MassPlan pl = mass_plan(p.rows, B, H, kv_len);
    const int splits = pl.splits;
    p.part = splits > 1 ? (float*)workspace : nullptr;
    const int64_t row_tiles = (p.rows + attn::MASS_ROWS - 1) / attn::MASS_ROWS;
    p.rows_per_split = (row_tiles + splits - 1) / splits * attn::MASS_ROWS;
    const int64_t work = B * H * pl.tiles * splits;
    HN_REQUIRE(work <= 0x3fffffffLL, HN_E_ARG, "hn_attn_key_mass: too much work for one launch");
    p.B = B; p.tiles = (int)pl.tiles; p.work = (int)work;
    p.per_xcd = (int)((work + 7) / 8);
    const dim3 grid((unsigned)(8 * (int64_t)p.per_xcd));
    hipStream_t st = (hipStream_t)stream;
    if (fmt == HN_KV_FP8) {
        if (pl.kb == 4) attn::key_mass_kernel<HN_KV_FP8, 4><<<grid, 256, 0, st>>>(p);
        else attn::key_mass_kernel<HN_KV_FP8, 1><<<grid, 256, 0, st>>>(p);
    } else {
        if (pl.kb == 4) attn::key_mass_kernel<HN_KV_INT8, 4><<<grid, 256, 0, st>>>(p);
        else attn::key_mass_kernel<HN_KV_INT8, 1><<<grid, 256, 0, st>>>(p);
    }
    const int rc = check_launch("hn_attn_key_mass");
    if (rc != HN_OK || splits == 1) return rc;
    attn::key_mass_sum_kernel<<<dim3((unsigned)((kv_len + 255) / 256), (unsigned)(B * H)), 256, 0, st>>>(p, splits);
    return check_launch("hn_attn_key_mass (sum)");
}
