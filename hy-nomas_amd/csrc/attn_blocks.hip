// Attention over chosen blocks of a quantized KV cache, and the weight that
// each cached key draws (gfx950).
//
//   hn_attn_kv_blocks: O = softmax(Q K^T scale) V and the rows' log-sum-exp, over
//     the keys of the blocks that a list names for each run of queries (without a
//     list: every cached key), then the bf16 tail.
//   hn_attn_key_mass:  mass[t] = sum over query rows of exp(s(row, t) - lse(row)).
//
// K, V = bf16(code * scale), as in attn_fp8kv.hip.
#include "attn_pages.h"
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
// Inf or NaN) meets a zero probability. The denominator is 0 only for a row without a
// key; a NaN that a row meets stays in it, and so in output and log-sum-exp. Bound by
// the vector work (dequantization, exponentials) beside the products and by waits at
// the two barriers a tile: 10800 queries x 24 heads, runs of 128, over 128 of 1350
// random blocks and a 10800-token tail 3.07-3.2 ms, 0.79-0.82 PFLOP/s; the same list
// for every run is 10 % faster (L2), the tail alone runs at 0.89, dense attention of 8
// waves at 0.95-1.0.
struct BlockParams : Params {
    const int32_t* idx;    // null: all blocks
    int64_t is0, is1, is2;
    int top_k, shift;      // block = 64 << shift tokens
    int64_t block;
    int64_t q_block, runs, B;
    int G;                 // query heads per cached head; H counts cached heads
    float* lse;            // [B, H G, Lq]
    const int32_t* lens;   // of pages: the sequences' tokens
    const int32_t* q_start;  // as in PageParams
    int pages;
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

// A list's entries, 64 at a time in a register (lane i: entry 64 chunk + i), so that an
// entry is a lane read: loaded entry by entry, each would wait for every load issued
// before it, the prefetched codes among them.
struct ListReader {
    const int32_t* list;
    int k, chunk, held;
    HN_DEVICE ListReader(const int32_t* l, int top_k) : list(l), k(top_k), chunk(-1), held(0) {}
    HN_DEVICE int operator()(int i) {  // entry i < k, the same for the whole wave
        if ((i >> 6) != chunk) {
            chunk = i >> 6;
            held = list[min(64 * chunk + (int)(threadIdx.x & 63), k - 1)];
        }
        return __builtin_amdgcn_readlane(held, i & 63);
    }
};

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

//
// PAGED: idx is a page table [B, top_k], block a page, and sequence b's tokens are the
// first lens[b] that its pages hold, in their order; a tile lies in one page and its loads
// go through descriptors of its own rows. The part of a tile past the length reads as zeros.
// It serves 33 to 128 rows, and more over short sequences (where, and what the others take:
// pages_plan). CAUSAL: no tail, and query i sees tokens below seen_before + i.
template <int FMT, bool MASK, bool PAGED = false, bool CAUSAL = false>
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
    const uint32_t rr = (uint32_t)(qvalid ? row : rows - 1), G = (uint32_t)p.G;
    const int64_t qi = i0 + rr / G, hq = h * p.G + rr % G;

    bf16x8 qf[8];
    {
        const uint16_t* src = p.q + b * p.qs0 + qi * p.qs1 + hq * p.qs2 + half * 8;
#pragma unroll
        for (int sl = 0; sl < 8; ++sl)
            qf[sl] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(src + 16 * sl));
    }

    const int32_t* list = p.idx ? p.idx + b * p.is0 + h * p.is1 + run * p.is2 : nullptr;
    const int kv_len = PAGED ? __builtin_amdgcn_readfirstlane(seq_len(p.lens, b, p.top_k, p.shift + 6)) : (int)p.kv_len;
    int lim = 0, lim_all = 0, lim_end = kv_len;  // CAUSAL: tokens that this row, every row and any row sees
    if constexpr (CAUSAL) {
        const int before = seen_before(p, b, kv_len), last = (int)rows - 1;
        lim = min(before + (int)qi, kv_len);
        lim_all = min(before + qt * BQ / p.G, kv_len);
        lim_end = max(min(before + min(qt * BQ + BQ - 1, last) / p.G, kv_len), 0);
    }
    const int n_cache = list && !PAGED ? list_length(list, p.top_k) << p.shift : (lim_end + BKV - 1) / BKV;
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

    // Loads go through descriptors that span the (b, h) rows of the cache [0, kv_len)
    // and of the tail: a tile is a 32-bit byte offset in them, and rows past their
    // ends read as zeros. A span of 2^31 bytes or more is replaced by the tile's own
    // rows, tile by tile.
    const bool span_ok = !PAGED && p.kv_len > 0 && (p.kv_len - 1) * p.cs1 + D < ((int64_t)1 << 31) &&
                         ((p.kv_len - 1) * p.ss1 + 1) * 4 < ((int64_t)1 << 31);
    const bool tail_ok = (p.cur_len * p.us1 + D) * 2 < ((int64_t)1 << 31);
    TileBase src = tile_base(p, b, h, 0, span_ok ? (int)p.kv_len : 0);
    auto tail_rsrc = [&](const uint16_t* base, int64_t first, int64_t rows) __attribute__((always_inline)) {
        return tile_rsrc(base + b * p.us0 + h * p.us2 + first * p.us1, rows > 0 ? ((rows - 1) * p.us1 + D) * 2 : 0);
    };
    const int64_t tail_rows = tail_ok ? p.cur_len : 0;
    __amdgpu_buffer_rsrc_t tk = tail_rsrc(p.kcur, 0, tail_rows), tv = tail_rsrc(p.vcur, 0, tail_rows);

    // Tile t: keys that exist, and where its loads start: code and scale offsets, its
    // first key in the validity bytes. Past the last tile, and for a list entry past
    // the last block: no key, and offsets past every span.
    struct Place {
        uint32_t co, so;
        int count, first;
    };
    constexpr uint32_t NOWHERE = 0x80000000u;
    ListReader reader(list, p.top_k);
    auto entry = [&](int t) __attribute__((always_inline)) {  // list entry of cache tile t
        if constexpr (PAGED) return t < n_cache && t < t_end ? scalar_ints(list)[t >> p.shift] : -1;
        return list && t < n_cache && t < t_end ? reader(t >> p.shift) : 0;
    };
    const int cur_len = (int)p.cur_len, entries = PAGED ? p.pages : (kv_len + (BKV << p.shift) - 1) >> (6 + p.shift);
    const uint32_t cs1 = (uint32_t)p.cs1, ss1 = (uint32_t)p.ss1 * 4u, us1 = (uint32_t)p.us1 * 2u;
    auto cache_place = [&](int t, int e) __attribute__((always_inline)) {
        Place g;
        const bool there = t < n_cache && t < t_end && (PAGED ? (uint32_t)e < (uint32_t)entries : e < entries);
        g.first = !there ? 0 : list && !PAGED ? ((e << p.shift) + (t & ((1 << p.shift) - 1))) * BKV : t * BKV;
        const int left = there ? kv_len - g.first : 0;
        g.count = left >= BKV ? BKV : left > 0 ? left : 0;
        g.co = g.count > 0 ? (uint32_t)g.first * cs1 : NOWHERE;
        g.so = g.count > 0 ? (uint32_t)g.first * ss1 : NOWHERE;
        if (!span_ok && g.count > 0) {
            if constexpr (PAGED) {
                src = tile_base(p, e, h, (t & ((1 << p.shift) - 1)) * BKV, g.count);
            } else {
                src = tile_base(p, b, h, g.first, g.count);
                src.mk = p.kvalid ? p.kvalid + b * p.kvs : nullptr;
            }
            g.co = g.so = 0;
        }
        return g;
    };
    auto tail_count = [&](int t) __attribute__((always_inline)) {
        const int left = t < t_end ? cur_len - (t - n_cache) * BKV : 0;
        return left >= BKV ? BKV : left > 0 ? left : 0;
    };
    auto tail_place = [&](int t) __attribute__((always_inline)) {
        Place g;
        g.first = (t - n_cache) * BKV;
        g.count = tail_count(t);
        g.co = g.count > 0 ? (uint32_t)g.first * us1 : NOWHERE;
        g.so = 0;
        if (!tail_ok && g.count > 0) {
            tk = tail_rsrc(p.kcur, g.first, g.count);
            tv = tail_rsrc(p.vcur, g.first, g.count);
            g.co = 0;
        }
        return g;
    };
    // The keys of a tile that take part: existing and (MASK) valid.
    auto word_of = [&](int count, const uint8_t* st) __attribute__((always_inline)) {
        const uint64_t all = count >= BKV ? ALL_KEYS : (1ull << count) - 1;
        return tile_mask<MASK>(st) & all;
    };
    // Half kb of cache tile t, its keys' word and largest logit: without those that take no part.
    auto masked = [&](f32x16& x, int t, int kb, uint64_t word, float mx) __attribute__((always_inline)) {
        if constexpr (CAUSAL)
            if ((t + 1) * BKV > lim_all) return mask_raw(x, kb, half, lim - t * BKV, word);
        const uint32_t w = (uint32_t)(word >> (32 * kb));
        return w == ~0u ? mx : mask_word(x, w);
    };
    const uint32_t ka_off = col * KROW + 16 * half;
    const uint32_t va_off = K_BYTES + col * VTROW + 16 * half;
    CacheRegs<NW> regs;
    regs.s = 0.0f;
    const LaneOffs<NW> lo = lane_offsets<NW>(p);
    auto fetch_k = [&](const Place& g) __attribute__((always_inline)) {
        load_k<NW, MASK>(lo, regs, src, g.count, g.co, g.so, g.first);
    };

    if (t_end > t_begin) {
        f32x16 sa, sb;
        float mxa, mxb;
        uint64_t mw;
        int count, next_count;  // existing keys of tiles t and t + 1
        TailRegs<NW> tr;
        const TailOffs<NW> to = tail_offsets<NW>(p);
        auto fetch_tail_k = [&](const Place& g) __attribute__((always_inline)) {
            load_tail_span_k<NW, MASK>(p, b, to, tk, g.co, g.first, g.first + g.count, tr);
        };
        // ---- prologue: tile t_begin to stage 0, the codes of the next to registers
        if (t_begin < n_cache) {
            const Place g = cache_place(t_begin, entry(t_begin));
            count = g.count;
            fetch_k(g);
            load_v<NW>(lo, regs, src, g.co);
            __builtin_amdgcn_s_waitcnt(0);
            if (threadIdx.x < 2 * BKV) sbuf[threadIdx.x] = regs.s;
            store_mask<NW, MASK>(regs, smem);
            __syncthreads();
            float ks[Shape<NW>::KU];
            k_scales<NW>(sbuf, ks);
            float4 vs = v_scales(sbuf);
            if constexpr (MASK) {
                const uint64_t word = word_of(count, smem);
                if (word != ALL_KEYS) clear_masked_v(regs, vs, word);
            }
            uint32_t kd[4];
            float vp[Shape<NW>::VD];
            uint32_t vd[2 * Shape<NW>::VD];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                store_k_part<FMT, NW>(regs, smem, i, ks, kd);
                store_v_part<FMT, NW>(regs.v, smem + K_BYTES, i, vs, vp, vd);
            }
        } else {
            const Place g = tail_place(t_begin);
            count = g.count;
            fetch_tail_k(g);
            load_tail_span_v<NW>(to, tv, g.co, tr);
            store_tail_k<NW, MASK>(tr, smem);
            if constexpr (MASK) {
                __syncthreads();
                const uint64_t word = word_of(count, smem);
                if (word != ALL_KEYS) clear_masked_v(tr, word);
            }
            store_tail_v<NW>(tr, smem);
        }
        {
            const Place g = cache_place(t_begin + 1, entry(t_begin + 1));
            next_count = t_begin + 1 < n_cache ? g.count : tail_count(t_begin + 1);
            fetch_k(g);
            load_v<NW>(lo, regs, src, g.co);
        }
        __builtin_amdgcn_s_waitcnt(0);
        if (threadIdx.x < 2 * BKV) sbuf[SB_FLOATS + threadIdx.x] = regs.s;
        __syncthreads();
        mw = word_of(count, smem);
        sa = s_block(smem + ka_off, qf);
        mxa = masked(sa, t_begin, 0, mw, raw_max(sa));
        int t = t_begin;
        int e2 = entry(t + 2);
        // ---- cache tiles, and the step into the tail
        for (; t < t_end && t < n_cache; ++t) {
            const int u = t - t_begin;
            const uint8_t* st = smem + (u & 1) * STAGE;
            uint8_t* nst = smem + ((u & 1) ^ 1) * STAGE;
            const float* nsb = sbuf + ((u & 1) ^ 1) * SB_FLOATS;
            const Place g2 = cache_place(t + 2, e2);
            e2 = entry(t + 3);
            f16x8 pf[2];
            // half 0
            rebase_high(mxa, c, run_, o);
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
            mxb = masked(sb, t, 1, mw, mxb);
            const bool tail_next = t + 1 < t_end && t + 1 >= n_cache;
            if (tail_next) {  // once: the tail's first tile, loaded on the spot
                fetch_tail_k(tail_place(t + 1));
                store_tail_k<NW, MASK>(tr, nst);
            }
            fetch_k(g2);
            __syncthreads();
            // half 1 (on the last tile the S block of "tile t + 1" reads stale LDS; its
            // result is never used)
            const uint64_t mwn = word_of(next_count, nst);
            rebase_high(mxb, c, run_, o);
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
            mxa = masked(sa, t + 1, 0, mwn, mxa);
            if (tail_next) {
                load_tail_span_v<NW>(to, tv, tail_place(t + 1).co, tr);
                if constexpr (MASK)
                    if (mwn != ALL_KEYS) clear_masked_v(tr, mwn);
                store_tail_v<NW>(tr, nst);
            }
            if (threadIdx.x < 2 * BKV) sbuf[(u & 1) * SB_FLOATS + threadIdx.x] = regs.s;
            load_v<NW>(lo, regs, src, g2.co);
            __syncthreads();
            next_count = t + 2 < n_cache ? g2.count : tail_count(t + 2);
            mw = mwn;
        }
        // ---- tail tiles
        if (t < t_end) {
            {
                const Place g = tail_place(t + 1);
                fetch_tail_k(g);
                load_tail_span_v<NW>(to, tv, g.co, tr);
            }
            for (; t < t_end; ++t) {
                const int u = t - t_begin;
                const uint8_t* st = smem + (u & 1) * STAGE;
                uint8_t* nst = smem + ((u & 1) ^ 1) * STAGE;
                f16x8 pf[2];
                rebase_high(mxa, c, run_, o);
                sb = step_a_lse(sa, c, run_.nm, run_.l, pf, st + ka_off + 32 * KROW, qf);
                mxb = step_b_with(pf, st + va_off, 0, o, sb, [&](int i) __attribute__((always_inline)) {
                    if (i & 1) store_tail_k_part<NW>(tr, nst, i >> 2, (i >> 1) & 1);
                });
                store_tail_mask<NW, MASK>(tr, nst);
                if ((uint32_t)(mw >> 32) != ~0u) mxb = mask_word(sb, (uint32_t)(mw >> 32));
                const Place g2 = tail_place(t + 2);
                fetch_tail_k(g2);
                __syncthreads();
                const uint64_t mwn = word_of(tail_count(t + 1), nst);  // (past the end: unused)
                if constexpr (MASK)
                    if (mwn != ALL_KEYS) clear_masked_v(tr, mwn);
                rebase_high(mxb, c, run_, o);
                sa = step_a_lse(sb, c, run_.nm, run_.l, pf, nst + ka_off, qf);
                mxa = step_b_with(pf, st + va_off, 1, o, sa, [&](int i) __attribute__((always_inline)) {
                    store_tail_v_part<NW>(tr, nst, i);
                });
                if ((uint32_t)mwn != ~0u) mxa = mask_word(sa, (uint32_t)mwn);
                load_tail_span_v<NW>(to, tv, g2.co, tr);
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
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
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
    if (half == 0) p.lse[at] = l != 0.0f ? (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f : -INFINITY;
}

// ---------------------------------------------------------------------------
// Runs of 33 to 64 rows: two row blocks of 32, and the two 32-key halves of a tile go to
// different waves (wave w: rows 32 (w % 2) .., keys 32 (w / 2) ..), so that four waves
// share each tile's dequantization. A wave has one half a tile to compute, so K runs
// two tiles ahead of its use by the PV product and V one: while tile t's probabilities
// are formed (beside S of t + 1) and multiplied, V of t + 1 goes to the other stage and
// K of t + 2 to this one, whose K was last read a tile ago; one barrier a tile. The two
// halves of a row's keys meet at the end. Scales travel four tiles ahead of V. Bound by
// the latency of the codes' loads (a tile is computed in less). At 254 to 256 VGPRs the
// registers are full, and the masked forms spill (12 bytes a lane in fp8, 20 in int8).
// 777 queries x 24 heads in runs of 64 over 24 int8 blocks of 128 with holes and a
// 777-token tail 139 us + 8.6 us of merge. Calls (merge included) against
// attn_blocks_kernel, whose waves are half idle: that one 149 against 170 us (fp8 without
// holes 129 against 136), runs of 48 162 against 190, of 33 240 against 258; a single run
// of 33 or 64 rows, 64 lists x 4096 keys 37.6 against 37.5 and 40.9 against 40.2, 64 x
// 32768 200 against 224 and 209 against 228, but 64 x 1024 22.3 against 20.5 and 25.5
// against 23.6: short lists pay for its longer prologue.
template <int FMT, bool MASK>
__global__ __launch_bounds__(256, 2) void attn_half_kernel(BlockParams p) {
    constexpr int NW = 4;
    __shared__ __attribute__((aligned(16))) uint8_t smem[2 * STAGE + 4 * SB_FLOATS * 4];
    float* const sbuf = reinterpret_cast<float*>(smem + 2 * STAGE);  // scales of tile t at (t % 4) SB_FLOATS
    const int id = blockIdx.x;
    const int w = (id & 7) * p.per_xcd + (id >> 3);
    if (w >= p.work) return;
    // the splits of a run, then the runs of a head
    int x = w;
    const int split = x % p.splits;
    x /= p.splits;
    const int64_t run = x % p.runs;
    x /= (int)p.runs;
    const int64_t h = x % p.H, b = x / p.H;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5, kb = wave >> 1;
    const int64_t i0 = run * p.q_block;
    const int64_t queries = p.Lq - i0 < p.q_block ? p.Lq - i0 : p.q_block;
    const int rows = (int)(queries * p.G), row = 32 * (wave & 1) + col;
    const bool qvalid = row < rows;
    const int rr = qvalid ? row : rows - 1;
    const int64_t qi = i0 + rr / p.G, hq = h * p.G + rr % p.G;
    bf16x8 qf[8];
    {
        const uint16_t* src = p.q + b * p.qs0 + qi * p.qs1 + hq * p.qs2 + half * 8;
#pragma unroll
        for (int sl = 0; sl < 8; ++sl)
            qf[sl] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(src + 16 * sl));
    }
    const int32_t* list = p.idx ? p.idx + b * p.is0 + h * p.is1 + run * p.is2 : nullptr;
    const int kv_len = (int)p.kv_len, cur_len = (int)p.cur_len, entries = (kv_len + (BKV << p.shift) - 1) >> (6 + p.shift);
    const int n_cache = list ? list_length(list, p.top_k) << p.shift : (kv_len + BKV - 1) / BKV;
    const int n_all = n_cache + (cur_len + BKV - 1) / BKV;
    const int t_begin = (int)((int64_t)n_all * split / p.splits), t_end = (int)((int64_t)n_all * (split + 1) / p.splits);
    f32x16 o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[i][v] = 0.0f;
    Run run_{-INFINITY, 0.0f, 0.0f};
    const float c = p.scale_log2;

    // Tiles as in attn_blocks_kernel: descriptors over the cache's and the tail's rows,
    // replaced by a tile's own where a span passes 2^31 bytes.
    const bool span_ok = p.kv_len > 0 && (p.kv_len - 1) * p.cs1 + D < ((int64_t)1 << 31) &&
                         ((p.kv_len - 1) * p.ss1 + 1) * 4 < ((int64_t)1 << 31);
    const bool tail_ok = (p.cur_len * p.us1 + D) * 2 < ((int64_t)1 << 31);
    auto tail_rsrc = [&](const uint16_t* base, int64_t first, int64_t n) __attribute__((always_inline)) {
        return tile_rsrc(base + b * p.us0 + h * p.us2 + first * p.us1, n > 0 ? ((n - 1) * p.us1 + D) * 2 : 0);
    };
    const TileBase span = tile_base(p, b, h, 0, span_ok ? kv_len : 0);
    const __amdgpu_buffer_rsrc_t tks = tail_rsrc(p.kcur, 0, tail_ok ? cur_len : 0),
                                 tvs = tail_rsrc(p.vcur, 0, tail_ok ? cur_len : 0);
    const uint32_t cs1 = (uint32_t)p.cs1, ss1 = (uint32_t)p.ss1 * 4u, us1 = (uint32_t)p.us1 * 2u;
    constexpr uint32_t NOWHERE = 0x80000000u;
    ListReader reader(list, p.top_k);
    struct Tile {
        int first, count;
    };
    auto tile_of = [&](int t) __attribute__((always_inline)) {
        Tile g{0, 0};
        if (t >= t_end) return g;
        int left;
        if (t < n_cache) {
            const int e = list ? reader(t >> p.shift) : 0;
            const bool there = e < entries;
            g.first = !there ? 0 : list ? ((e << p.shift) + (t & ((1 << p.shift) - 1))) * BKV : t * BKV;
            left = there ? kv_len - g.first : 0;
        } else {
            g.first = (t - n_cache) * BKV;
            left = cur_len - g.first;
        }
        g.count = left >= BKV ? BKV : left > 0 ? left : 0;
        return g;
    };
    auto word_of = [&](int count, const uint8_t* st) __attribute__((always_inline)) {
        const uint64_t all = count >= BKV ? ALL_KEYS : (1ull << count) - 1;
        return tile_mask<MASK>(st) & all;
    };
    const uint32_t ka_off = (32 * kb + col) * KROW + 16 * half;
    const uint32_t va_off = K_BYTES + col * VTROW + 16 * half;
    CacheRegs<NW> regs;
    regs.s = 0.0f;
    regs.mk = 0u;
    TailRegs<NW> tr;
    tr.mk = 0u;
    const LaneOffs<NW> lo = lane_offsets<NW>(p);
    const TailOffs<NW> to = tail_offsets<NW>(p);
    // K codes and validity of a tile (of the cache or the tail, CT) to registers; V codes;
    // the scales
    auto fetch_k = [&](auto ct, const Tile& g) __attribute__((always_inline)) {
        if constexpr (decltype(ct)::value) {
            TileBase src = span;
            uint32_t co = g.count > 0 ? (uint32_t)g.first * cs1 : NOWHERE;
            if (!span_ok) {
                src = tile_base(p, b, h, g.first, g.count);
                co = 0;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
                regs.k[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(src.k, lo.k[i] + co, 0, 0));
            if constexpr (MASK)
                if (wave == 2)
                    regs.mk = lane < g.count ? (p.kvalid ? (uint32_t)p.kvalid[b * p.kvs + g.first + lane] : 1u) : 0u;
        } else {
            const bool own = !tail_ok;
            load_tail_span_k<NW, MASK>(p, b, to, own ? tail_rsrc(p.kcur, g.first, g.count) : tks,
                                       own ? 0u : g.count > 0 ? (uint32_t)g.first * us1 : NOWHERE, g.first,
                                       g.first + g.count, tr);
        }
    };
    auto fetch_v = [&](auto ct, const Tile& g) __attribute__((always_inline)) {
        if constexpr (decltype(ct)::value) {
            TileBase src = span;
            uint32_t co = g.count > 0 ? (uint32_t)g.first * cs1 : NOWHERE;
            if (!span_ok) {
                src = tile_base(p, b, h, g.first, g.count);
                co = 0;
            }
            load_v<NW>(lo, regs, src, co);
        } else {
            const bool own = !tail_ok;
            load_tail_span_v<NW>(to, own ? tail_rsrc(p.vcur, g.first, g.count) : tvs,
                                 own ? 0u : g.count > 0 ? (uint32_t)g.first * us1 : NOWHERE, tr);
        }
    };
    auto fetch_s = [&](const Tile& g, bool cache) __attribute__((always_inline)) {
        if (wave >= 2 || !cache) return;
        TileBase src = span;
        uint32_t so_ = g.count > 0 ? (uint32_t)g.first * ss1 : NOWHERE;
        if (!span_ok) {
            src = tile_base(p, b, h, g.first, g.count);
            so_ = 0;
        }
        const __amdgpu_buffer_rsrc_t sr = wave == 0 ? src.ks : src.vs;
        regs.s = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(sr, lo.s + so_, 0, 0));
    };
    auto put_s = [&](int t) __attribute__((always_inline)) {
        if (threadIdx.x < 2 * BKV) sbuf[(t & 3) * SB_FLOATS + threadIdx.x] = regs.s;
    };
    auto scales = [&](int t) __attribute__((always_inline)) { return sbuf + (t & 3) * SB_FLOATS; };
    const auto cache_c = std::integral_constant<bool, true>{};
    const auto tail_c = std::integral_constant<bool, false>{};
    auto stage = [&](int t) __attribute__((always_inline)) { return smem + ((t - t_begin) & 1) * STAGE; };

    if (t_end > t_begin) {
        // ---- prologue: K of t_begin and t_begin + 1 and V of t_begin in LDS, V of t_begin + 1
        // and K of t_begin + 2 in registers, scales up to t_begin + 3
        auto store_k_now = [&](auto ct, int t) __attribute__((always_inline)) {
            uint8_t* st = stage(t);
            if constexpr (decltype(ct)::value) {
                store_mask<NW, MASK>(regs, st);
                float ks[2];
                k_scales<NW>(scales(t), ks);
                uint32_t kd[4];
#pragma unroll
                for (int i = 0; i < 8; ++i) store_k_part<FMT, NW>(regs, st, i, ks, kd);
            } else {
                store_tail_k<NW, MASK>(tr, st);
            }
        };
        Tile g0 = tile_of(t_begin), g1 = tile_of(t_begin + 1), g2 = tile_of(t_begin + 2), g3 = tile_of(t_begin + 3);
        fetch_s(g0, t_begin < n_cache);
        put_s(t_begin);
        fetch_s(g1, t_begin + 1 < n_cache);
        put_s(t_begin + 1);
        fetch_s(g2, t_begin + 2 < n_cache);
        put_s(t_begin + 2);
        if (t_begin < n_cache) fetch_k(cache_c, g0);
        else fetch_k(tail_c, g0);
        __syncthreads();
        if (t_begin < n_cache) store_k_now(cache_c, t_begin);
        else store_k_now(tail_c, t_begin);
        if (t_begin + 1 < n_cache) {
            fetch_k(cache_c, g1);
            store_k_now(cache_c, t_begin + 1);
        } else {
            fetch_k(tail_c, g1);
            store_k_now(tail_c, t_begin + 1);
        }
        __syncthreads();
        const uint64_t mw0 = word_of(g0.count, stage(t_begin));
        if (t_begin < n_cache) {
            fetch_v(cache_c, g0);
            float4 vs = v_scales(scales(t_begin));
            if constexpr (MASK)
                if (mw0 != ALL_KEYS) clear_masked_v(regs, vs, mw0);
            float vp[8];
            uint32_t vd[16];
#pragma unroll
            for (int i = 0; i < 8; ++i) store_v_part<FMT, NW>(regs.v, stage(t_begin) + K_BYTES, i, vs, vp, vd);
        } else {
            fetch_v(tail_c, g0);
            if constexpr (MASK)
                if (mw0 != ALL_KEYS) clear_masked_v(tr, mw0);
            store_tail_v<NW>(tr, stage(t_begin));
        }
        fetch_s(g3, t_begin + 3 < n_cache);
        if (t_begin + 1 < n_cache) fetch_v(cache_c, g1);
        else fetch_v(tail_c, g1);
        if (t_begin + 2 < n_cache) fetch_k(cache_c, g2);
        else fetch_k(tail_c, g2);
        f32x16 s = s_block(stage(t_begin) + ka_off, qf);
        float mx = raw_max(s);
        if ((uint32_t)(mw0 >> (32 * kb)) != ~0u) mx = mask_word(s, (uint32_t)(mw0 >> (32 * kb)));
        __syncthreads();
        // ---- tile t; KT, VT: K of t + 2, V of t + 1 are the cache's
        auto iterate = [&](auto kt, auto vt_, int t) __attribute__((always_inline)) {
            constexpr bool KT = decltype(kt)::value, VT = decltype(vt_)::value;
            uint8_t* st = stage(t);
            uint8_t* nst = stage(t + 1);
            const Tile g4 = tile_of(t + 4);
            f16x8 pf[2];
            rebase_high(mx, c, run_, o);
            f32x16 sn = step_a_lse(s, c, run_.nm, run_.l, pf, nst + ka_off, qf);
            const uint64_t mwn = word_of(g1.count, nst);
            float4 vs = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float ks[2] = {0.0f, 0.0f};
            if constexpr (VT) vs = v_scales(scales(t + 1));
            if constexpr (KT) k_scales<NW>(scales(t + 2), ks);
            if constexpr (MASK)
                if (mwn != ALL_KEYS) {
                    if constexpr (VT) clear_masked_v(regs, vs, mwn);
                    else clear_masked_v(tr, mwn);
                }
            uint32_t kd[4], vd[16];
            float vp[8];
            mx = step_b_with(pf, st + va_off, kb, o, sn, [&](int i) __attribute__((always_inline)) {
                if constexpr (VT) store_v_part<FMT, NW>(regs.v, nst + K_BYTES, i, vs, vp, vd);
                else store_tail_v_part<NW>(tr, nst, i);
                if constexpr (KT) store_k_part<FMT, NW>(regs, st, i, ks, kd);
                else if (i & 1) store_tail_k_part<NW>(tr, st, i >> 2, (i >> 1) & 1);
            });
            if constexpr (KT) store_mask<NW, MASK>(regs, st);
            else store_tail_mask<NW, MASK>(tr, st);
            if ((uint32_t)(mwn >> (32 * kb)) != ~0u) mx = mask_word(sn, (uint32_t)(mwn >> (32 * kb)));
            s = sn;
            put_s(t + 3);
            fetch_s(g4, t + 4 < n_cache);
            if (t + 2 < n_cache) fetch_v(cache_c, g2);
            else fetch_v(tail_c, g2);
            if (t + 3 < n_cache) fetch_k(cache_c, g3);
            else fetch_k(tail_c, g3);
            __syncthreads();
            g1 = g2;
            g2 = g3;
            g3 = g4;
        };
        int t = t_begin;
        for (; t < t_end && t + 2 < n_cache; ++t) iterate(cache_c, cache_c, t);
        for (; t < t_end && t + 1 < n_cache; ++t) iterate(tail_c, cache_c, t);
        for (; t < t_end; ++t) iterate(tail_c, tail_c, t);
    }
    // ---- the two key halves of a row meet: waves 2 and 3 pass theirs through LDS
    float l = run_.l + __shfl_xor(run_.l, 32, 64), m = run_.m;
    constexpr int PITCH = D + 4;
    float* so = reinterpret_cast<float*>(smem);  // [64][PITCH], then [64][2]
    float* sml = so + 64 * PITCH;
    __syncthreads();
    if (kb == 1) {
        float* dst = so + row * PITCH;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int vq = 0; vq < 4; ++vq)
                *reinterpret_cast<float4*>(dst + db * 32 + vq * 8 + half * 4) =
                    make_float4(o[db][vq * 4], o[db][vq * 4 + 1], o[db][vq * 4 + 2], o[db][vq * 4 + 3]);
        if (half == 0) {
            sml[2 * row] = m;
            sml[2 * row + 1] = l;
        }
    }
    __syncthreads();
    if (kb == 1 || !qvalid) return;
    const float m1 = sml[2 * row], top = fmaxf(m, m1), base = top == -INFINITY ? 0.0f : top;
    const float a0 = __builtin_amdgcn_exp2f(m - base), a1 = __builtin_amdgcn_exp2f(m1 - base);
    l = l * a0 + sml[2 * row + 1] * a1;
    m = top;
    const int64_t hqs = p.H * p.G, at = (b * hqs + hq) * p.Lq + qi;
    const int64_t slot = (int64_t)split * p.B * hqs * p.Lq + at;
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    uint16_t* dst = p.out + b * p.os0 + qi * p.os1 + hq * p.os2;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int vq = 0; vq < 4; ++vq) {
            const int d = db * 32 + vq * 8 + half * 4;
            const float4 y = *reinterpret_cast<const float4*>(so + row * PITCH + d);
            const float4 v = make_float4(o[db][vq * 4] * a0 + y.x * a1, o[db][vq * 4 + 1] * a0 + y.y * a1,
                                         o[db][vq * 4 + 2] * a0 + y.z * a1, o[db][vq * 4 + 3] * a0 + y.w * a1);
            if (p.splits > 1) *reinterpret_cast<float4*>(p.ws_o + slot * D + d) = v;
            else *reinterpret_cast<uint2*>(dst + d) = make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
        }
    if (half != 0) return;
    if (p.splits > 1) *reinterpret_cast<float2*>(p.ws_ml + slot * 2) = make_float2(m, l);
    else p.lse[at] = l != 0.0f ? (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f : -INFINITY;
}

// ---------------------------------------------------------------------------
// One row a run (single tokens of ungrouped heads). The read of the keys is the whole
// cost and a matrix tile would hold one row of 32, so the products run on the vector
// unit, without LDS or barriers in the loop: 8 lanes hold a key (16 dims each, one
// 16-byte load of K and of V), a wave reads 8 keys per load and has a whole 64-key
// tile in flight. K^ enters as packed bf16 (v_dot2_f32_bf16 onto fp32), probabilities
// and V^ as fp32. Each lane group runs an online softmax of its own keys; the 8 groups
// of a wave, the 4 waves and the splits meet at the end. Calls (merge included) against
// attn_waves_kernel: 64 lists x 1024 keys 10.5 against 13.8 us, x 4096 23.9 against 28.5,
// x 32768 135 against 153 (4.1 TB/s); 77 runs of 24 heads over 48 blocks and a 77-token
// tail 318 against 300.
struct RowState {
    float m, l, o[16];
};

HN_DEVICE float dpp_add8(float v) {  // sum over the 8 lanes of an aligned group
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0xB1, 0xf, 0xf, true));
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x4E, 0xf, 0xf, true));
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x141, 0xf, 0xf, true));
    return v;
}

// bf16(code * s) of a lane's 16 codes, as 8 packed words.
template <int FMT>
HN_DEVICE void held16(const uint4& x, float s, uint32_t (&w)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const f32x2 f = codes2_f32<FMT>(word(x, i >> 1), i & 1);
        w[i] = pack_bf16(f[0] * s, f[1] * s);
    }
}

// The group's logit (log2 units) of one key.
HN_DEVICE float row_logit(const uint32_t (&k)[8], const uint32_t (&q)[8], float c, bool there) {
    float a = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        a = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, k[i]), __builtin_bit_cast(bf16x2, q[i]), a, false);
    a = dpp_add8(a);
    return there ? a * c : -INFINITY;
}

// The running maximum takes in N keys' logits; O and l follow it.
template <int N>
HN_DEVICE void row_rebase(const float (&s)[N], RowState& f) {
    float mx = f.m;
#pragma unroll
    for (int e = 0; e < N; ++e) mx = fmaxf(mx, s[e]);
    const float a = mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(f.m - mx);
    f.m = mx;
    f.l *= a;
#pragma unroll
    for (int d = 0; d < 16; ++d) f.o[d] *= a;
}

HN_DEVICE void row_add(float s, const uint32_t (&v)[8], bool there, RowState& f) {
    const float p = there ? __builtin_amdgcn_exp2f(s - f.m) : 0.0f;
    f.l += p;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        f.o[2 * i] = __builtin_fmaf(p, bf16_lo(v[i]), f.o[2 * i]);
        f.o[2 * i + 1] = __builtin_fmaf(p, bf16_hi(v[i]), f.o[2 * i + 1]);
    }
}

template <int FMT>
__global__ __launch_bounds__(256, 2) void attn_row_kernel(BlockParams p) {
    __shared__ float so[4][D], sml[4][2];
    const int id = blockIdx.x;
    const int w = (id & 7) * p.per_xcd + (id >> 3);
    if (w >= p.work) return;
    // heads fastest, then the splits of a row
    const int64_t h = w % p.H;
    int x = w / (int)p.H;
    const int split = x % p.splits;
    x /= p.splits;
    const int64_t run = x % p.runs, b = x / p.runs, i = run * p.q_block;  // (G = 1: head h, query i)
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int piece = lane & 7, grp = lane >> 3;
    uint32_t q[8];
    {
        const uint4* src = reinterpret_cast<const uint4*>(p.q + b * p.qs0 + i * p.qs1 + h * p.qs2 + 16 * piece);
        const uint4 y0 = src[0], y1 = src[1];
        q[0] = y0.x; q[1] = y0.y; q[2] = y0.z; q[3] = y0.w;
        q[4] = y1.x; q[5] = y1.y; q[6] = y1.z; q[7] = y1.w;
    }
    const int32_t* list = p.idx ? p.idx + b * p.is0 + h * p.is1 + run * p.is2 : nullptr;
    const int kv_len = (int)p.kv_len, cur_len = (int)p.cur_len;
    const int entries = (kv_len + (BKV << p.shift) - 1) >> (6 + p.shift);
    const int n_cache = list ? list_length(list, p.top_k) << p.shift : (kv_len + BKV - 1) / BKV;
    const int n_all = n_cache + (cur_len + BKV - 1) / BKV;
    ListReader reader(list, p.top_k);
    const float c = p.scale_log2;
    RowState f;
    f.m = -INFINITY;
    f.l = 0.0f;
#pragma unroll
    for (int d = 0; d < 16; ++d) f.o[d] = 0.0f;
    // tiles of 64 keys, dealt to the waves of all splits in turn
    for (int t = split * 4 + wave; t < n_all; t += 4 * p.splits) {
        if (t < n_cache) {
            int first = t * BKV, left = kv_len - first;
            if (list) {
                const int e = reader(t >> p.shift);
                first = e < entries ? ((e << p.shift) + (t & ((1 << p.shift) - 1))) * BKV : 0;
                left = e < entries ? kv_len - first : 0;
            }
            if (left <= 0) continue;
            const int64_t base = b * p.cs0 + first * p.cs1 + h * p.cs2 + 16 * piece;
            uint4 kx[8], vx[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)  // (a key past the end reads the last one)
                kx[e] = *reinterpret_cast<const uint4*>(p.kc + base + min(8 * e + grp, left - 1) * p.cs1);
            // this lane's scales and validity: key 8 piece + grp, read by its group in step `piece`
            const int mine = min(8 * piece + grp, left - 1);
            const int64_t sa = b * p.ss0 + (first + mine) * p.ss1 + h * p.ss2;
            const float ks = p.ks[sa], vs = p.vs[sa];
            int ok = 8 * piece + grp < left;
            if (p.kvalid) ok &= p.kvalid[b * p.kvs + first + mine] != 0;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                vx[e] = *reinterpret_cast<const uint4*>(p.vc + base + min(8 * e + grp, left - 1) * p.cs1);
            float s[8];
            uint32_t there = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                uint32_t kw[8];
                held16<FMT>(kx[e], __shfl(ks, (lane & 56) + e, 64), kw);
                const bool in = __shfl(ok, (lane & 56) + e, 64) != 0;
                there |= (uint32_t)in << e;
                s[e] = row_logit(kw, q, c, in);
            }
            row_rebase<8>(s, f);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool in = (there >> e) & 1u;
                uint32_t vw[8];
                // (what a masked key holds must not meet its zero probability)
                const float sv = __shfl(vs, (lane & 56) + e, 64);
                held16<FMT>(in ? vx[e] : make_uint4(0u, 0u, 0u, 0u), in ? sv : 0.0f, vw);
                row_add(s[e], vw, in, f);
            }
        } else {
            const int first = (t - n_cache) * BKV, left = cur_len - first;
            for (int e = 0; e < 8 && 8 * e < left; ++e) {
                const int j = first + min(8 * e + grp, left - 1);
                const bool in = 8 * e + grp < left && (!p.uvalid || p.uvalid[b * p.uvs + j] != 0);
                const int64_t at = b * p.us0 + j * p.us1 + h * p.us2 + 16 * piece;
                const uint4 *kp = reinterpret_cast<const uint4*>(p.kcur + at), *vp = reinterpret_cast<const uint4*>(p.vcur + at);
                const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
                const uint4 a0 = in ? kp[0] : zero, a1 = in ? kp[1] : zero, b0 = in ? vp[0] : zero, b1 = in ? vp[1] : zero;
                const uint32_t kw[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
                const uint32_t vw[8] = {b0.x, b0.y, b0.z, b0.w, b1.x, b1.y, b1.z, b1.w};
                const float s[1] = {row_logit(kw, q, c, in)};
                row_rebase<1>(s, f);
                row_add(s[0], vw, in, f);
            }
        }
    }
    // The 8 groups of the wave: common maximum, then the dims are dealt out while the
    // groups add up (lane xor 32, 16, 8), each lane ending with two dims.
    {
        float m = f.m;
#pragma unroll
        for (int off = 8; off < 64; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
        const float a = f.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(f.m - m);
        float l = f.l * a;
#pragma unroll
        for (int off = 8; off < 64; off <<= 1) l += __shfl_xor(l, off, 64);
        float v8[8], v4[4];
#pragma unroll
        for (int d = 0; d < 8; ++d) {
            const float keep = (grp & 4 ? f.o[8 + d] : f.o[d]) * a, give = (grp & 4 ? f.o[d] : f.o[8 + d]) * a;
            v8[d] = keep + __shfl_xor(give, 32, 64);
        }
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            const float keep = grp & 2 ? v8[4 + d] : v8[d], give = grp & 2 ? v8[d] : v8[4 + d];
            v4[d] = keep + __shfl_xor(give, 16, 64);
        }
        const int d0 = 16 * piece + 8 * (grp >> 2) + 4 * ((grp >> 1) & 1) + 2 * (grp & 1);
#pragma unroll
        for (int d = 0; d < 2; ++d) {
            const float keep = grp & 1 ? v4[2 + d] : v4[d], give = grp & 1 ? v4[d] : v4[2 + d];
            so[wave][d0 + d] = keep + __shfl_xor(give, 8, 64);
        }
        if (lane == 0) {
            sml[wave][0] = m;
            sml[wave][1] = l;
        }
    }
    __syncthreads();
    if (threadIdx.x >= D) return;
    // the 4 waves, a thread a dim
    const int d = threadIdx.x;
    const float m = fmaxf(fmaxf(sml[0][0], sml[1][0]), fmaxf(sml[2][0], sml[3][0]));
    const float base = m == -INFINITY ? 0.0f : m;
    float l = 0.0f, v = 0.0f;
#pragma unroll
    for (int wv = 0; wv < 4; ++wv) {
        const float a = __builtin_amdgcn_exp2f(sml[wv][0] - base);
        l = __builtin_fmaf(sml[wv][1], a, l);
        v = __builtin_fmaf(so[wv][d], a, v);
    }
    const int64_t slot = (b * p.H + h) * p.Lq + i;
    if (p.splits > 1) {
        const int64_t part = (int64_t)split * p.B * p.H * p.Lq + slot;
        p.ws_o[part * D + d] = v;
        if (d == 0) *reinterpret_cast<float2*>(p.ws_ml + part * 2) = make_float2(m, l);
    } else {
        p.out[b * p.os0 + i * p.os1 + h * p.os2 + d] = (uint16_t)f32_to_bf16_bits(l != 0.0f ? v / l : 0.0f);
        if (d == 0) p.lse[slot] = l != 0.0f ? (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f : -INFINITY;
    }
}

// ---------------------------------------------------------------------------
// Up to 32 rows a run: one matrix column block holds them all, so the waves of a
// workgroup share the keys instead of the rows. Every wave takes 32-key blocks of its
// own, without barriers: K codes go from global memory to MFMA operands in registers
// (lane half: 64 contiguous dims, which the Q operand matches), V^ passes through the
// wave's own LDS tile to be transposed ([dim][key], as attn_tiles.h). While a block is
// computed the next one's codes are in flight to a second set of registers. The waves
// and the splits meet at the end. Bound by the read of the keys and, where each wave has
// few blocks, by a fixed 8 us (launch, first loads, meeting): 64 lists x 4096 keys, 4
// rows each (69 MB) 25 us, 64 x 8192 35 us (5.8 TB/s for the second half). It fills 256
// VGPRs and spills 10 (44 bytes a lane). Calls (merge included) against attn_half_kernel
// and attn_blocks_kernel: 4 rows 28.4, 34.6, 35.5 us; 32 rows 31.8, 36.8, 36.8; 777
// queries x 24 heads in runs of 32 over 48 blocks and the tail 145, 229, 229.
constexpr int WV_ROW = 80;                       // V^T row: 32 fp16 keys + 16 B
constexpr int WV_GROUP = 16 * WV_ROW + 64;       // 16 rows + 64 B (writes of 4 row groups fall in different banks)
constexpr int WV_BYTES = 8 * WV_GROUP;
constexpr int WO_PITCH = D + 4;                  // floats
constexpr int WAVES_SMEM = 4 * 32 * WO_PITCH * 4;  // the partial outputs of 4 waves (over the V^T tiles)
static_assert(4 * WV_BYTES <= WAVES_SMEM, "V^T tiles fit");

HN_DEVICE int wv_row(int dim) { return (dim >> 4) * WV_GROUP + (dim & 15) * WV_ROW; }

struct WaveRegs {  // codes of a 32-key block
    uint4 k[4];    // key col, dims 64 half ..
    uint4 v[4];    // keys quad_key(lane % 8, j), dims 16 (lane / 8) ..
    float ks, vs;  // of key col
    int left;      // keys that exist, from key 0 on (<= 0: none)
    uint32_t ok;   // of key col: valid
};

template <int FMT>
__global__ __launch_bounds__(256, 2) void attn_waves_kernel(BlockParams p) {
    __shared__ __attribute__((aligned(16))) uint8_t smem[WAVES_SMEM];
    __shared__ float sml[4][32][2];
    const int id = blockIdx.x;
    const int w = (id & 7) * p.per_xcd + (id >> 3);
    if (w >= p.work) return;
    // Lists: the splits of a run, then the runs of a head. Whole cache: heads fastest,
    // which share the lines of a key range's scales.
    int64_t h, run, b;
    int split, x = w;
    if (p.idx) {
        split = x % p.splits;
        x /= p.splits;
        run = x % p.runs;
        x /= (int)p.runs;
        h = x % p.H;
        b = x / p.H;
    } else {
        h = x % p.H;
        x /= (int)p.H;
        split = x % p.splits;
        x /= p.splits;
        run = x % p.runs;
        b = x / p.runs;
    }
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5, qd = lane & 7, dg = lane >> 3;
    const int64_t i0 = run * p.q_block;
    const int64_t queries = p.Lq - i0 < p.q_block ? p.Lq - i0 : p.q_block;
    const int rows = (int)(queries * p.G);  // 1 .. 32
    uint8_t* const vt = smem + wave * WV_BYTES;
    bf16x8 qf[8];
    {
        const int r = col < rows ? col : rows - 1;
        const uint16_t* src = p.q + b * p.qs0 + (i0 + r / p.G) * p.qs1 + (h * p.G + r % p.G) * p.qs2 + 64 * half;
#pragma unroll
        for (int sl = 0; sl < 8; ++sl) qf[sl] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(src + 8 * sl));
    }
    const int32_t* list = p.idx ? p.idx + b * p.is0 + h * p.is1 + run * p.is2 : nullptr;
    const int kv_len = (int)p.kv_len, cur_len = (int)p.cur_len;
    const int entries = (kv_len + (BKV << p.shift) - 1) >> (6 + p.shift);
    const int sh32 = p.shift + 1;  // block = 32 << sh32 tokens
    const int limit = list ? p.top_k << sh32 : (kv_len + 31) / 32;
    const int step = 4 * p.splits;
    ListReader reader(list, p.top_k);

    f32x16 o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[i][v] = 0.0f;
    Run run_{-INFINITY, 0.0f, 0.0f};
    const float c = p.scale_log2;

    // Loads through descriptors spanning the (b, h) rows of the cache, at 32-bit offsets
    // (rows past kv_len read as zeros); a span of 2^31 bytes or more is replaced by the
    // block's own rows, block by block.
    const uint32_t cs1 = (uint32_t)p.cs1, ss1 = (uint32_t)p.ss1 * 4u;
    const bool span_ok = p.kv_len > 0 && (p.kv_len - 1) * p.cs1 + D < ((int64_t)1 << 31) &&
                         ((p.kv_len - 1) * p.ss1 + 1) * 4 < ((int64_t)1 << 31);
    TileBase src = tile_base(p, b, h, 0, span_ok ? kv_len : 0);
    const uint32_t off_k = (uint32_t)col * cs1 + 64u * half, off_s = (uint32_t)col * ss1;
    uint32_t off_v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) off_v[j] = (uint32_t)quad_key(qd, j) * cs1 + 16u * dg;
    // Codes of cache block t < limit; a block without a key leaves `left` 0. (The first
    // loads do not wait for the list's length: what lies past its end is dropped
    // afterwards.)
    auto load = [&](int t, WaveRegs& r) __attribute__((always_inline)) {
        r.left = 0;
        if (t >= limit) return;
        int first = t * 32, left = kv_len - first;
        if (list) {
            const int e = reader(t >> sh32);
            const bool there = (uint32_t)e < (uint32_t)entries;
            first = there ? ((e << sh32) + (t & ((1 << sh32) - 1))) * 32 : 0;
            left = there ? kv_len - first : 0;
        }
        if (left <= 0) return;
        uint32_t co = (uint32_t)first * cs1, so_ = (uint32_t)first * ss1;
        if (!span_ok) {
            src = tile_base(p, b, h, first, min(left, 32));
            co = so_ = 0;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            r.k[e] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(src.k, off_k + co + 16 * e, 0, 0));
        r.ks = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(src.ks, off_s + so_, 0, 0));
        r.vs = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(src.vs, off_s + so_, 0, 0));
        r.ok = p.kvalid ? (uint32_t)p.kvalid[b * p.kvs + first + min(col, left - 1)] : 1u;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            r.v[j] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(src.v, off_v[j] + co, 0, 0));
        r.left = left;
    };
    // P and PV of a block whose V^T operands are vf (operand 4 tt + db).
    auto finish = [&](f32x16& s, uint32_t word, const f16x8 (&vf)[8]) __attribute__((always_inline)) {
        const float mx = word != ~0u ? mask_word(s, word) : raw_max(s);
        rebase_high(mx, c, run_, o);
        f16x8 pf[2];
        uint32_t x8[8];
        float l0 = 0.0f, l1 = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * i], c, run_.nm));
            const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * i + 1], c, run_.nm));
            x8[i] = pack_f16(p0, p1);
            l0 += p0;
            l1 += p1;
        }
        run_.l += l0 + l1;
        pf[0] = __builtin_bit_cast(f16x8, make_uint4(x8[0], x8[1], x8[2], x8[3]));
        pf[1] = __builtin_bit_cast(f16x8, make_uint4(x8[4], x8[5], x8[6], x8[7]));
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i & 3] = mfma_f16(vf[i], pf[i >> 2], o[i & 3]);
    };
    auto read_v = [&](f16x8 (&vf)[8]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) vf[i] = ld_f16x8(vt + wv_row(32 * (i & 3) + col) + 32 * (i >> 2) + 16 * half);
    };
    auto block = [&](WaveRegs& r) __attribute__((always_inline)) {
        // the keys that take part (asked for here: at the load it would wait for it)
        const uint32_t live = (uint32_t)__ballot(col < r.left && r.ok != 0u);
        if (live == 0) return;
        float vs[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) vs[j] = __shfl(r.vs, quad_key(qd, j), 64);
        if (live != ~0u) {  // what a masked key holds meets no product
            const uint32_t m = live >> quad_key(qd, 0);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool in = (m >> j) & 1u;
                r.v[j].x = in ? r.v[j].x : 0u;
                r.v[j].y = in ? r.v[j].y : 0u;
                r.v[j].z = in ? r.v[j].z : 0u;
                r.v[j].w = in ? r.v[j].w : 0u;
                vs[j] = in ? vs[j] : 0.0f;
            }
        }
        // Slot sl: K operand sl and its product, and V^ dims 16 dg + 2 sl, + 1 of the quad's
        // keys to the V^T tile.
        f32x16 s;
#pragma unroll
        for (int v = 0; v < 16; ++v) s[v] = 0.0f;
#pragma unroll
        for (int sl = 0; sl < 8; ++sl) {
            uint32_t d[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const f32x2 f = codes2_f32<FMT>(word(r.k[sl >> 1], 2 * (sl & 1) + (e >> 1)), e & 1);
                d[e] = pack_bf16(f[0] * r.ks, f[1] * r.ks);
            }
            s = mfma_bf16(__builtin_bit_cast(bf16x8, make_uint4(d[0], d[1], d[2], d[3])), qf[sl], s);
            f32x2 f[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f[j] = codes2_f32<FMT>(word(r.v[j], sl >> 1), sl & 1);
                f[j][0] *= vs[j];
                f[j][1] *= vs[j];
            }
#pragma unroll
            for (int e = 0; e < 2; ++e)
                *reinterpret_cast<uint2*>(vt + dg * WV_GROUP + (2 * sl + e) * WV_ROW + 8 * qd) =
                    make_uint2(pack_f16_of_bf16(f[0][e], f[1][e]), pack_f16_of_bf16(f[2][e], f[3][e]));
            __builtin_amdgcn_sched_barrier(0);
        }
        f16x8 vf[8];
        read_v(vf);
        finish(s, live, vf);
    };
    const int dealt = split * 4 + wave;  // blocks dealt, dealt + step, ..
    {
        int t = dealt;
        WaveRegs ra, rb;
        load(t, ra);
        load(t + step, rb);
        const int n_cache = list ? list_length(list, p.top_k) << sh32 : limit;
        while (t < n_cache) {
            block(ra);
            t += step;
            if (t >= n_cache) break;
            load(t + step, ra);
            block(rb);
            t += step;
            load(t + step, rb);
        }
    }
    // Tail blocks, dealt from the last wave on. One set of registers: the next block's V
    // is fetched once this one's is in LDS, its K once its logits are formed.
    const int n_tail = (cur_len + 31) / 32;
    if (step - 1 - dealt < n_tail) {
        uint4 kx[8], vx[4][2];
        bool ok = false;
        auto fetch_k = [&](int t) __attribute__((always_inline)) {
            const int first = t * 32, left = cur_len - first;
            if (left <= 0) return;
            const int mine = first + min(col, left - 1);
            const uint4* kp = reinterpret_cast<const uint4*>(p.kcur + b * p.us0 + mine * p.us1 + h * p.us2 + 64 * half);
#pragma unroll
            for (int sl = 0; sl < 8; ++sl) kx[sl] = kp[sl];
            ok = col < left && (!p.uvalid || p.uvalid[b * p.uvs + mine] != 0);
        };
        auto fetch_v = [&](int t) __attribute__((always_inline)) {
            const int first = t * 32, left = cur_len - first;
            if (left <= 0) return;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint4* vp = reinterpret_cast<const uint4*>(
                    p.vcur + b * p.us0 + (first + min(quad_key(qd, j), left - 1)) * p.us1 + h * p.us2 + 16 * dg);
                vx[j][0] = vp[0];
                vx[j][1] = vp[1];
            }
        };
        int t = step - 1 - dealt;
        fetch_k(t);
        fetch_v(t);
        for (; t < n_tail; t += step) {
            const uint32_t now = (uint32_t)__ballot(ok);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint32_t y[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    y[j] = word(vx[j][i >> 2], i & 3);
                    if (now != ~0u && !((now >> quad_key(qd, j)) & 1u)) y[j] = 0u;
                }
                uint8_t* dst = vt + dg * WV_GROUP + 2 * i * WV_ROW + 8 * qd;
                *reinterpret_cast<uint2*>(dst) = make_uint2(
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(bf16_lo(y[0]), bf16_lo(y[1]))),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(bf16_lo(y[2]), bf16_lo(y[3]))));
                *reinterpret_cast<uint2*>(dst + WV_ROW) = make_uint2(
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(bf16_hi(y[0]), bf16_hi(y[1]))),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(bf16_hi(y[2]), bf16_hi(y[3]))));
            }
            fetch_v(t + step);
            f32x16 s;
#pragma unroll
            for (int v = 0; v < 16; ++v) s[v] = 0.0f;
#pragma unroll
            for (int sl = 0; sl < 8; ++sl) s = mfma_bf16(__builtin_bit_cast(bf16x8, kx[sl]), qf[sl], s);
            fetch_k(t + step);
            f16x8 vf[8];
            read_v(vf);
            if (now != 0) finish(s, now, vf);
        }
    }
    // The four waves' partial results meet in LDS (over the V^T tiles).
    const float l = run_.l + __shfl_xor(run_.l, 32, 64);
    __syncthreads();
    float* so = reinterpret_cast<float*>(smem);
    if (col < rows) {
        float* dst = so + (wave * 32 + col) * WO_PITCH;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int vq = 0; vq < 4; ++vq)
                *reinterpret_cast<float4*>(dst + db * 32 + vq * 8 + half * 4) =
                    make_float4(o[db][vq * 4], o[db][vq * 4 + 1], o[db][vq * 4 + 2], o[db][vq * 4 + 3]);
        if (half == 0) {
            sml[wave][col][0] = run_.m;
            sml[wave][col][1] = l;
        }
    }
    __syncthreads();
    const int64_t hqs = p.H * p.G;
    for (int at = threadIdx.x; at < rows * (D / 4); at += 256) {
        const int r = at / (D / 4), d = (at % (D / 4)) * 4;
        float m = sml[0][r][0];
#pragma unroll
        for (int wv = 1; wv < 4; ++wv) m = fmaxf(m, sml[wv][r][0]);
        const float base = m == -INFINITY ? 0.0f : m;
        float den = 0.0f;
        float4 num = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int wv = 0; wv < 4; ++wv) {
            const float a = __builtin_amdgcn_exp2f(sml[wv][r][0] - base);
            const float4 y = *reinterpret_cast<const float4*>(so + (wv * 32 + r) * WO_PITCH + d);
            den = __builtin_fmaf(sml[wv][r][1], a, den);
            num.x = __builtin_fmaf(y.x, a, num.x);
            num.y = __builtin_fmaf(y.y, a, num.y);
            num.z = __builtin_fmaf(y.z, a, num.z);
            num.w = __builtin_fmaf(y.w, a, num.w);
        }
        const int64_t i = i0 + r / p.G, hq = h * p.G + r % p.G, slot = (b * hqs + hq) * p.Lq + i;
        if (p.splits > 1) {
            const int64_t part = (int64_t)split * p.B * hqs * p.Lq + slot;
            *reinterpret_cast<float4*>(p.ws_o + part * D + d) = num;
            if (d == 0) *reinterpret_cast<float2*>(p.ws_ml + part * 2) = make_float2(m, den);
        } else {
            const float inv = den != 0.0f ? 1.0f / den : 0.0f;
            *reinterpret_cast<uint2*>(p.out + b * p.os0 + i * p.os1 + hq * p.os2 + d) =
                make_uint2(pack_bf16(num.x * inv, num.y * inv), pack_bf16(num.z * inv, num.w * inv));
            if (d == 0) p.lse[slot] = den != 0.0f ? (m + __builtin_amdgcn_logf(den)) * 0.6931471805599453f : -INFINITY;
        }
    }
}

// Merge of the key splits, with the row's log-sum-exp: with M = max m_s,
// O = sum 2^(m_s - M) O_s / sum 2^(m_s - M) l_s. 32 threads a row, 4 dims each, eight
// splits' loads in flight; the order of the sums is that of the splits. 256 rows of 8
// splits 4.1 us (6.4 one load at a time), 18648 rows of 3 8.6 us.
__global__ __launch_bounds__(256) void blocks_combine_kernel(BlockParams p) {
    const int64_t hqs = p.H * p.G, rows = p.B * hqs * p.Lq;  // < 2^31
    const uint32_t r = blockIdx.x * 8 + (threadIdx.x >> 5);   // (b * Hq + hq) * Lq + i
    if (r >= rows) return;
    const int d = (threadIdx.x & 31) * 4;
    float M = -INFINITY, den = 0.0f;
    float4 num = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s0 = 0; s0 < p.splits; s0 += 8) {
        float2 ml[8];
        float4 ov[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int64_t at = (int64_t)min(s0 + e, p.splits - 1) * rows + r;
            ml[e] = *reinterpret_cast<const float2*>(p.ws_ml + at * 2);
            ov[e] = *reinterpret_cast<const float4*>(p.ws_o + at * D + d);
            if (s0 + e >= p.splits) ml[e] = make_float2(-INFINITY, 0.0f);  // (the last split again: no weight)
        }
        float top = M;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, ml[e].x);
        const float base = top == -INFINITY ? 0.0f : top, a = __builtin_amdgcn_exp2f(M - base);
        den *= a;
        num.x *= a; num.y *= a; num.z *= a; num.w *= a;
        M = top;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float wgt = __builtin_amdgcn_exp2f(ml[e].x - base);
            den = fmaf(wgt, ml[e].y, den);
            num.x = fmaf(wgt, ov[e].x, num.x);
            num.y = fmaf(wgt, ov[e].y, num.y);
            num.z = fmaf(wgt, ov[e].z, num.z);
            num.w = fmaf(wgt, ov[e].w, num.w);
        }
    }
    const uint32_t bh = r / (uint32_t)p.Lq, i = r - bh * (uint32_t)p.Lq, b = bh / (uint32_t)hqs, hq = bh - b * (uint32_t)hqs;
    const float inv = den != 0.0f ? 1.0f / den : 0.0f;
    *reinterpret_cast<uint2*>(p.out + b * p.os0 + i * p.os1 + hq * p.os2 + d) =
        make_uint2(pack_bf16(num.x * inv, num.y * inv), pack_bf16(num.z * inv, num.w * inv));
    if (d == 0) p.lse[r] = den != 0.0f ? (M + __builtin_amdgcn_logf(den)) * 0.6931471805599453f : -INFINITY;
}

// ---------------------------------------------------------------------------
// Key mass. A wave holds 32 KB keys as MFMA operands in registers; the query rows
// stream past them through LDS, 32 at a time. S = Q K^T puts one key per lane
// column, so a key's mass is a sum over the lane's own registers and one exchange
// with lane ^ 32 at the end; the rows' log-sum-exps come as four 16-byte LDS reads
// a tile. The MFMAs of one key block run beside the exponentials of the one before.
// One workgroup sees every row of its keys (or, split, its share of the rows, added
// in order afterwards), so no two add to one key and the result has one order.
// Bound by the exponentials beside the products, 3600 queries x 24 heads over
// 86400 keys 1.83 ms, 1.05 PFLOP/s (a large bf16 product reaches 1.39; one row per lane
// column, keys in registers, took 2.64 ms).
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
    int keys;               // of a workgroup of key_mass_few_kernel
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

    // This thread's 32 bytes of a query tile: row tid / 8, dims 16 (tid % 8) ..
    const int tr = tid >> 3, tu = tid & 7;
    const int64_t row0 = split * p.rows_per_split;
    const int64_t row1 = row0 + p.rows_per_split < p.rows ? row0 + p.rows_per_split : p.rows;
    uint4 x0, x1;
    float lse = INFINITY;
    // Row r of the next fetch: query head g of the group, query i, batch bb; each fetch
    // moves 32 rows on (steps dg, di, db with their carries; no division, and the ones
    // here in 32 bits).
    const uint32_t G = (uint32_t)p.G, Lq = p.Lq > 0 ? (uint32_t)p.Lq : 1u;
    int64_t r = row0 + tr;
    const uint32_t q0 = (uint32_t)r / G;
    uint32_t g = (uint32_t)r - q0 * G, i = q0 % Lq;
    int64_t bb = b * p.batches + q0 / Lq;
    const uint32_t dg = MASS_ROWS % G, di = (MASS_ROWS / G) % Lq, db = MASS_ROWS / G / Lq;
    auto fetch = [&]() {
        x0 = x1 = make_uint4(0u, 0u, 0u, 0u);
        lse = INFINITY;
        if (r < row1) {  // (the query does not wait for its log-sum-exp)
            const uint16_t* src = p.q + bb * p.qs0 + i * p.qs1 + (h * p.G + g) * p.qs2 + 16 * tu;
            x0 = reinterpret_cast<const uint4*>(src)[0];
            x1 = reinterpret_cast<const uint4*>(src)[1];
            lse = p.lse[(bb * p.H * p.G + h * p.G + g) * p.Lq + i];
        }
        r += MASS_ROWS;
        g += dg;
        i += di;
        bb += db;
        if (g >= G) {
            g -= G;
            ++i;
        }
        if (i >= Lq) {
            i -= Lq;
            ++bb;
        }
    };
    fetch();

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

    auto put = [&](int buf) {
        uint4* dst = reinterpret_cast<uint4*>(smem + buf * MASS_TILE + tr * KROW + 32 * tu);
        // a row without a finite log-sum-exp adds nothing, whatever it holds: exp2(0 - inf) = 0
        const bool counts = __builtin_fabsf(lse) < INFINITY;
        const uint32_t keep = counts ? ~0u : 0u;
        dst[0] = make_uint4(x0.x & keep, x0.y & keep, x0.z & keep, x0.w & keep);
        dst[1] = make_uint4(x1.x & keep, x1.y & keep, x1.z & keep, x1.w & keep);
        if (tu == 0) nl[buf][tr] = counts ? -lse * 1.4426950408889634f : -INFINITY;
    };
    float acc[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) acc[kb] = 0.0f;
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

// Up to 32 rows (single tokens): they are one MFMA operand, held in registers with their
// log-sum-exps while the keys stream past, 32 a wave at a time, without LDS or barriers;
// a block's codes go from global memory to operands while the next block's are in flight
// to a second set of registers. Bound by the read of the codes: 64
// heads x 32768 keys (293 MB), 4 rows each, 61 us, 4.8 TB/s (a copy reaches 5.1), where
// key_mass_kernel, one barrier and one short life a workgroup, took 81.
struct MassRegs {  // key col of a 32-key block
    uint4 y[4];    // dims 64 half ..
    float ks, before;
    uint32_t ok;   // valid (before: its prior mass)
};

template <int FMT>
__global__ __launch_bounds__(256, 4) void key_mass_few_kernel(MassParams p) {
    const int w = (int)(blockIdx.x & 7) * p.per_xcd + (int)(blockIdx.x >> 3);
    if (w >= p.work) return;
    const int64_t h = w % p.H;
    const int x = w / p.H, tile = x % p.tiles;
    const int64_t b = x / p.tiles;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    const int kv_len = (int)p.kv_len, first = tile * p.keys, last = kv_len - first < p.keys ? kv_len : first + p.keys;
    const float c = p.scale_log2;
    const uint8_t* const kc = p.kc + b * p.cs0 + h * p.cs2 + 64 * half;
    const float* const scales = p.ks + b * p.ss0 + h * p.ss2;
    const float* const prior = p.prior ? p.prior + b * p.ps0 + h * p.ps1 : nullptr;
    float* const mass = p.mass + (b * p.H + h) * p.kv_len;
    auto load = [&](int k0, MassRegs& r) __attribute__((always_inline)) {
        if (k0 >= last) return;
        const int64_t key = min(k0 + col, kv_len - 1);
        const uint4* src = reinterpret_cast<const uint4*>(kc + key * p.cs1);
#pragma unroll
        for (int e = 0; e < 4; ++e) r.y[e] = src[e];
        r.ks = scales[key * p.ss1];
        r.ok = p.valid ? (uint32_t)p.valid[b * p.vs + key] : 1u;
        r.before = prior && key < p.prior_len ? prior[key] : 0.0f;
    };
    int k0 = first + 32 * wave;
    MassRegs ra, rb;
    load(k0, ra);
    // row col of the query heads of this head's group: its dims 64 half .., its log-sum-exp
    bf16x8 qf[8];
    float nl = -INFINITY;
    {
        const uint32_t G = (uint32_t)p.G, Lq = p.Lq > 0 ? (uint32_t)p.Lq : 1u, q0 = (uint32_t)col / G, g = col - q0 * G;
        const uint32_t bb = q0 / Lq, i = q0 - bb * Lq;
        const int64_t qb = b * p.batches + bb, hq = h * p.G + g;
        const bool there = col < p.rows;
        const float lse = there ? p.lse[(qb * p.H * p.G + hq) * p.Lq + i] : INFINITY;
        // a row without a finite log-sum-exp adds nothing, whatever it holds: exp2(0 - inf) = 0
        const bool counts = __builtin_fabsf(lse) < INFINITY;
        const uint32_t keep = counts ? ~0u : 0u;
        if (counts) nl = -lse * 1.4426950408889634f;
        const uint16_t* src = p.q + qb * p.qs0 + i * p.qs1 + hq * p.qs2 + 64 * half;
#pragma unroll
        for (int sl = 0; sl < 8; ++sl) {
            uint4 y = make_uint4(0u, 0u, 0u, 0u);
            if (there) y = reinterpret_cast<const uint4*>(src)[sl];
            qf[sl] = __builtin_bit_cast(bf16x8, make_uint4(y.x & keep, y.y & keep, y.z & keep, y.w & keep));
        }
    }
    f32x16 n;  // row 8 (v / 4) + 4 half + v % 4
#pragma unroll
    for (int v = 0; v < 16; ++v) n[v] = __shfl(nl, 8 * (v >> 2) + 4 * half + (v & 3), 64);
    auto block = [&](int k0, MassRegs& r) __attribute__((always_inline)) {
        f32x16 s;
#pragma unroll
        for (int v = 0; v < 16; ++v) s[v] = 0.0f;
#pragma unroll
        for (int sl = 0; sl < 8; ++sl) {
            uint32_t d[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const f32x2 f = codes2_f32<FMT>(word(r.y[sl >> 1], 2 * (sl & 1) + (e >> 1)), e & 1);
                d[e] = pack_bf16(f[0] * r.ks, f[1] * r.ks);
            }
            s = mfma_bf16(qf[sl], __builtin_bit_cast(bf16x8, make_uint4(d[0], d[1], d[2], d[3])), s);
            __builtin_amdgcn_sched_barrier(0);
        }
        float a0 = 0.0f, a1 = 0.0f;
#pragma unroll
        for (int v = 0; v < 16; v += 2) {
            a0 += __builtin_amdgcn_exp2f(__builtin_fmaf(s[v], c, n[v]));
            a1 += __builtin_amdgcn_exp2f(__builtin_fmaf(s[v + 1], c, n[v + 1]));
        }
        const float half_sum = a0 + a1, sum = half_sum + __shfl_xor(half_sum, 32, 64);
        // (the column of an invalid key, whatever it holds, is dropped)
        if (half == 0 && k0 + col < last) mass[k0 + col] = r.ok != 0u ? r.before + sum : r.before;
    };
    while (k0 < last) {
        load(k0 + 128, rb);
        block(k0, ra);
        k0 += 128;
        if (k0 >= last) break;
        load(k0 + 128, ra);
        block(k0, rb);
        k0 += 128;
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

// Which kernel a run's rows take: one row attn_row_kernel, up to 32 attn_waves_kernel,
// up to 64 attn_half_kernel, more attn_blocks_kernel (both sides of each border are
// measured at the kernels).
enum class BlocksKernel { ROW, WAVES, HALF, TILES };

struct BlocksPlan {
    BlocksKernel kernel;
    int64_t runs, q_tiles, work;
    int splits;
};

// Key splits. Two workgroups fit a CU; with sp splits the launch takes
// ceil(work sp / 2 CUs) rounds of workgroups, each worth its tiles (64 keys; a
// workgroup of the first two kernels works on four at a time) and a fixed part (the
// list, the first loads, the end), and the merge reads and writes every row sp times.
// In units of a tile of a full round (2.7 us measured in attn_blocks_kernel; the other
// kernels' tiles were not measured apart): the split with the least of it is taken, each
// keeping at least 4 tiles.
static BlocksPlan blocks_plan(int64_t B, int64_t Lq, int64_t Hq, int64_t H, int64_t kv_len, int64_t cur_len,
                              int64_t top_k, int64_t block, int64_t q_block) {
    constexpr double FIXED = 2.0, MERGE = 1e-4;  // per workgroup; per row and split (1 KB at 4 TB/s)
    BlocksPlan pl;
    pl.runs = (Lq - 1) / q_block + 1;
    const int64_t rows = (q_block < Lq ? q_block : Lq) * (Hq / H);
    const int64_t listed = top_k >= 0 ? top_k * (block / attn::BKV) : (kv_len + attn::BKV - 1) / attn::BKV;
    const int64_t tiles = listed + (cur_len + attn::BKV - 1) / attn::BKV;
    pl.kernel = rows == 1    ? BlocksKernel::ROW
                : rows <= 32 ? BlocksKernel::WAVES
                : rows <= 64 ? BlocksKernel::HALF
                             : BlocksKernel::TILES;
    pl.q_tiles = pl.kernel == BlocksKernel::TILES ? (rows + attn::Shape<4>::BQ - 1) / attn::Shape<4>::BQ : 1;
    pl.work = B * H * pl.runs * pl.q_tiles;
    pl.splits = 1;
    const int64_t slots = 2LL * device_cus(), at_once = rows <= 32 ? 4 : 1;
    double best = 1e30;
    for (int64_t sp = 1; sp <= 64 && (sp == 1 || 4 * sp <= tiles + 3) && (sp == 1 || pl.work * sp <= 8 * slots); ++sp) {
        const double rounds = (double)((pl.work * sp + slots - 1) / slots);
        const double cost = rounds * (FIXED + (double)tiles / (double)(at_once * sp)) +
                            (sp > 1 ? MERGE * (double)sp * (double)(B * Hq * Lq) : 0.0);
        if (cost < best) {
            best = cost;
            pl.splits = (int)sp;
        }
    }
    return pl;
}

template <int FMT>
static void launch_blocks(BlocksKernel kernel, bool mask, const attn::BlockParams& p, dim3 grid, hipStream_t st) {
    if (kernel == BlocksKernel::ROW) attn::attn_row_kernel<FMT><<<grid, 256, 0, st>>>(p);
    else if (kernel == BlocksKernel::WAVES) attn::attn_waves_kernel<FMT><<<grid, 256, 0, st>>>(p);
    else if (kernel == BlocksKernel::HALF && mask) attn::attn_half_kernel<FMT, true><<<grid, 256, 0, st>>>(p);
    else if (kernel == BlocksKernel::HALF) attn::attn_half_kernel<FMT, false><<<grid, 256, 0, st>>>(p);
    else if (mask) attn::attn_blocks_kernel<FMT, true><<<grid, 256, 0, st>>>(p);
    else attn::attn_blocks_kernel<FMT, false><<<grid, 256, 0, st>>>(p);
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
        HN_REQUIRE(curs[3] == 1 && curs[0] % 8 == 0 && curs[1] % 8 == 0 && curs[2] % 8 == 0 && curs[0] >= 0 &&
                       curs[1] >= 0 && curs[1] <= 0xffffffLL && curs[2] >= 0,
                   HN_E_ARG, "hn_attn_kv_blocks: tail strides must be multiples of 8, below 2^24 per token");
        HN_REQUIRE(aligned(kcur, 16) && aligned(vcur, 16), HN_E_ARG, "hn_attn_kv_blocks: tail misaligned");
    }
    if (B == 0 || Lq == 0) return HN_OK;
    HN_REQUIRE(q && out && lse, HN_E_ARG, "hn_attn_kv_blocks: null q/out/lse");
    const BlocksPlan pl = blocks_plan(B, Lq, Hq, H, kv_len, cur_len, idx ? top_k : -1, block, q_block);
    const int64_t need = pl.splits > 1 ? (int64_t)pl.splits * B * Hq * Lq * (attn::D + 2) * (int64_t)sizeof(float) : 0;
    HN_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned(workspace, 16))), HN_E_ARG,
               "hn_attn_kv_blocks: workspace smaller than hn_attn_kv_blocks_workspace_size() or misaligned");
    const int64_t work = pl.work * pl.splits;
    HN_REQUIRE(work <= 0x3fffffffLL && pl.runs <= 0x3fffffffLL && B * Hq * Lq <= 0x7fffffffLL, HN_E_ARG,
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
    if (fmt == HN_KV_FP8) launch_blocks<HN_KV_FP8>(pl.kernel, mask, p, grid, st);
    else launch_blocks<HN_KV_INT8>(pl.kernel, mask, p, grid, st);
    const int rc = check_launch("hn_attn_kv_blocks");
    if (rc != HN_OK || pl.splits == 1) return rc;
    attn::blocks_combine_kernel<<<(unsigned)((B * Hq * Lq + 7) / 8), 256, 0, st>>>(p);
    return check_launch("hn_attn_kv_blocks (combine)");
}

// Tiles of 128 rows over pages: the plan is that of as many tokens as the table can name.
static BlocksPlan page_tiles_plan(int64_t B, int64_t Lq, int64_t Hq, int64_t H, int64_t max_len, int64_t cur_len) {
    // (65 rows at least: the tile kernel whatever their number)
    const int64_t rows = Lq * (Hq / H), as_rows = rows < 65 ? (65 + Hq / H - 1) / (Hq / H) : Lq;
    BlocksPlan pl = blocks_plan(B, as_rows, Hq, H, max_len, cur_len, -1, 64, as_rows);
    pl.q_tiles = (rows + attn::Shape<4>::BQ - 1) / attn::Shape<4>::BQ;
    pl.work = B * H * pl.q_tiles;
    return pl;
}

static int64_t page_tiles_bytes(const BlocksPlan& pl, int64_t rows) {
    return pl.splits > 1 ? pl.splits * rows * (attn::D + 2) * (int64_t)sizeof(float) : 0;
}

int64_t hn::page_tiles_workspace(int64_t B, int64_t Lq, int64_t Hq, int64_t H, int64_t max_len, int64_t cur_len) {
    return page_tiles_bytes(page_tiles_plan(B, Lq, Hq, H, max_len, cur_len), B * Hq * Lq);
}

int hn::launch_page_tiles(const attn::PageParams& a, int fmt, void* workspace, hipStream_t st) {
    const int64_t Hq = (int64_t)a.H * a.G, rows = a.B * Hq * a.Lq;
    const BlocksPlan pl = page_tiles_plan(a.B, a.Lq, Hq, a.H, (int64_t)a.width << a.shift, a.cur_len);
    const int64_t work = pl.work * pl.splits;
    HN_REQUIRE(work <= 0x3fffffffLL && rows <= 0x7fffffffLL, HN_E_ARG, "hn_attn_kv_pages: too much work for one launch");
    attn::BlockParams p = {};
    p.q = a.q; p.out = a.out; p.lse = a.lse;
    p.kc = a.kc; p.vc = a.vc; p.ks = a.ks; p.vs = a.vs;
    p.kcur = a.kcur; p.vcur = a.vcur;
    p.uvalid = a.uvalid; p.uvs = a.uvs;
    p.qs0 = a.qs0; p.qs1 = a.qs1; p.qs2 = a.qs2;
    p.os0 = a.os0; p.os1 = a.os1; p.os2 = a.os2;
    p.cs0 = a.cs0; p.cs1 = a.cs1; p.cs2 = a.cs2;
    p.ss0 = a.ss0; p.ss1 = a.ss1; p.ss2 = a.ss2;
    p.us0 = a.us0; p.us1 = a.us1; p.us2 = a.us2;
    p.Lq = a.Lq; p.H = a.H; p.G = a.G; p.B = a.B; p.cur_len = a.cur_len;
    p.scale_log2 = a.scale_log2;
    p.fmt = fmt;
    p.idx = a.table; p.is0 = a.ts0;
    p.top_k = a.width;
    p.lens = a.lens; p.q_start = a.q_start; p.pages = a.pages;
    p.block = (int64_t)1 << a.shift;
    p.shift = a.shift - 6;
    p.q_block = a.Lq; p.runs = 1;
    p.q_tiles = (int)pl.q_tiles; p.splits = pl.splits;
    p.work = (int)work;
    p.per_xcd = (int)((work + 7) / 8);
    if (pl.splits > 1) {
        p.ws_o = (float*)workspace;
        p.ws_ml = (float*)workspace + pl.splits * rows * attn::D;
    }
    const dim3 grid((unsigned)(8 * (int64_t)p.per_xcd));
    if (fmt == HN_KV_FP8) {
        if (a.causal) attn::attn_blocks_kernel<HN_KV_FP8, false, true, true><<<grid, 256, 0, st>>>(p);
        else if (p.uvalid) attn::attn_blocks_kernel<HN_KV_FP8, true, true><<<grid, 256, 0, st>>>(p);
        else attn::attn_blocks_kernel<HN_KV_FP8, false, true><<<grid, 256, 0, st>>>(p);
    } else {
        if (a.causal) attn::attn_blocks_kernel<HN_KV_INT8, false, true, true><<<grid, 256, 0, st>>>(p);
        else if (p.uvalid) attn::attn_blocks_kernel<HN_KV_INT8, true, true><<<grid, 256, 0, st>>>(p);
        else attn::attn_blocks_kernel<HN_KV_INT8, false, true><<<grid, 256, 0, st>>>(p);
    }
    const int rc = check_launch("hn_attn_kv_pages");
    if (rc != HN_OK || pl.splits == 1) return rc;
    attn::blocks_combine_kernel<<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(p);
    return check_launch("hn_attn_kv_pages (join)");
}

// Plan of the key mass. Up to 32 rows: key_mass_few_kernel (KB 0), with as many keys a
// workgroup as leave eight workgroups a CU, 128 to 1024. More: 512 keys per workgroup (KB
// 4: each row tile read from LDS once for four key blocks), or 128 (KB 1) where 512 would
// not fill the device twice over; where even these fall short (a short cache, many
// queries) the rows are split, each split writes its sums and a second kernel adds them in
// order. KB 1 against KB 4, 24 heads: 3600 queries over 5500 keys (264 workgroups of 512)
// 217 against 225 us, 10800 keys (528) 358 against 332, 86400 2493 against 1787; with few
// rows the border would lie higher, 64 queries over 11000 keys 18.6 against 21.0, 86400
// 106 against 107.
struct MassPlan {
    int kb, splits, keys;
    int64_t tiles;
};

static MassPlan mass_plan(int64_t rows, int64_t B, int64_t H, int64_t kv_len) {
    const int64_t target = 2LL * device_cus();
    if (rows <= attn::MASS_ROWS) {
        const int64_t steps = B * H * ((kv_len + 127) / 128) / (4 * target);
        const int keys = 128 * (int)(steps < 1 ? 1 : steps > 8 ? 8 : steps);
        return MassPlan{0, 1, keys, (kv_len + keys - 1) / keys};
    }
    MassPlan pl{4, 1, 0, (kv_len + 511) / 512};
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
    HN_REQUIRE(p.rows <= 0x3fffffffLL, HN_E_ARG, "hn_attn_key_mass: too many query rows");
    const MassPlan pl = mass_plan(p.rows, B, H, kv_len);
    const int splits = pl.splits;
    p.part = splits > 1 ? (float*)workspace : nullptr;
    const int64_t row_tiles = (p.rows + attn::MASS_ROWS - 1) / attn::MASS_ROWS;
    p.rows_per_split = (row_tiles + splits - 1) / splits * attn::MASS_ROWS;
    const int64_t work = B * H * pl.tiles * splits;
    HN_REQUIRE(work <= 0x3fffffffLL, HN_E_ARG, "hn_attn_key_mass: too much work for one launch");
    p.B = B; p.tiles = (int)pl.tiles; p.keys = pl.keys; p.work = (int)work;
    p.per_xcd = (int)((work + 7) / 8);
    const dim3 grid((unsigned)(8 * (int64_t)p.per_xcd));
    hipStream_t st = (hipStream_t)stream;
    if (pl.kb == 0) {
        if (fmt == HN_KV_FP8) attn::key_mass_few_kernel<HN_KV_FP8><<<grid, 256, 0, st>>>(p);
        else attn::key_mass_few_kernel<HN_KV_INT8><<<grid, 256, 0, st>>>(p);
    } else if (fmt == HN_KV_FP8) {
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
