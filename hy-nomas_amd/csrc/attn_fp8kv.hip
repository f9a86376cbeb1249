// Block-causal chunk attention over an FP8 (or INT8-compat) KV cache, gfx950.
//
//   O = softmax(Q K^T * scale) V,   K, V = code * per-(token, head) scale
//
// Work decomposition: one workgroup = NW waves = 32 NW queries of one (batch,
// head); each wave owns 32 queries (one 32-column MFMA block). Two shapes:
// 4 waves (128 queries, two workgroups per CU) and 8 waves (256 queries, one
// per CU); both put 2 waves on each SIMD, and the 8-wave shape dequantizes
// each K/V tile once for twice the queries. Keys stream through LDS in tiles
// of 64. Each tile is dequantized once per workgroup as it is written to LDS,
// to the reference's own dequantized values: K = bf16(code * k_scale) and
// V = bf16(code * v_scale) (fp32 product, rounded to nearest even), so the
// MFMAs consume exactly the K/V the reference attends over, and no per-key
// scale is needed in the compute loop. The optional unquantized tail (the
// current chunk's bf16 K/V) is copied into the same LDS formats.
//
// Per 32-key block the wave computes S^T = K Q^T with
// v_mfma_f32_32x32x16_bf16: the MFMA output puts one query per lane column,
// so a block's max is lane-local. The running max m moves only when a block's
// logits pass m + 8 (one exchange with lane ^ 32 then makes it the pair's
// exact max): probabilities stay <= 2^8, and the common path has no
// cross-lane step. The row sum (of the fp16 probabilities, v_dot2) stays
// lane-local until the end. P^T is packed to fp16 in
// registers and is the B operand of O^T += V^T P^T (v_mfma_f32_32x32x16_f16).
// fp16 probabilities round at 2^-11 relative instead of bf16's 2^-8; V^T is
// held as the fp16 form of its bf16 value, which is the same number (a bf16
// value in fp16's normal range is exactly representable; fp16 subnormals
// round below 2^-24 and magnitudes past 65504 saturate). V is kept
// transposed in LDS ([dim][key], keys of each 16-key slice in the order of
// the P^T registers), so each V^T operand is one 16-byte LDS read.
//
// The loop is software-pipelined over half tiles (32-key blocks) so that each
// wave's MFMAs run beside independent VALU work of its own (see step_a /
// step_b).
//
// Mask: key position p is visible to query position r iff p / chunk <= r / chunk
// (chunk <= 0: all visible), and, in the MASK instantiation, iff the key's
// validity byte is non-zero (padded text keys, holes in the cached history:
// the kv_mask of nomas_cpt.py:611-685). Tiles wholly beyond the last query's
// chunk are never visited; tiles wholly visible to every query of the
// workgroup skip the per-element test.
#include <mutex>

#include "attn_tiles.h"

namespace hn {
namespace attn {

template <int FMT, int NW, bool MASK>
__global__ __launch_bounds__(64 * NW, 8 / NW) void attn_fp8kv_kernel(Params p) {
    constexpr int BQ = Shape<NW>::BQ;
    constexpr int NS = stages<NW>();
    __shared__ __attribute__((aligned(16))) uint8_t smem[smem_bytes<NW>()];
    float* const sbuf = reinterpret_cast<float*>(smem + NS * STAGE);  // [2][128]

    // XCD-aware work order: workgroup ids are dealt round-robin to the 8 XCDs,
    // so id % 8 picks a contiguous range of work items.
    //  * No key split: items run (b, h, query tile) with the tile fastest, so
    //    the query tiles of the same few heads share an XCD's L2 while they
    //    stream those heads' K/V.
    //  * Key splits: items run (b, query tile, split, h) with the head
    //    fastest, so an XCD holds whole key ranges of every head. A token's
    //    per-head scales are adjacent ([B, cap, H, 1]): the heads of one key
    //    range then share each scale sector in one L2, where a head-major
    //    order had every XCD fetch every sector for its few heads.
    const int id = blockIdx.x;
    const int w = (id & 7) * p.per_xcd + (id >> 3);
    if (w >= p.work) return;
    int split, qt;
    int64_t h, b;
    if (p.splits > 1) {
        h = w % p.H;
        const int ws = w / (int)p.H;
        split = ws % p.splits;
        const int wt = ws / p.splits;
        qt = wt % p.q_tiles;
        b = wt / p.q_tiles;
    } else {
        split = 0;
        qt = w % p.q_tiles;
        h = (w / p.q_tiles) % p.H;
        b = w / (p.q_tiles * (int)p.H);
    }

    const int lane = threadIdx.x & 63;
    const int wave = threadIdx.x >> 6;
    const int col = lane & 31, half = lane >> 5;
    const int64_t row = (int64_t)qt * BQ + wave * QW + col;  // this lane's query row
    const bool qvalid = row < p.Lq;
    const int64_t qrow = qvalid ? row : p.Lq - 1;
    const int64_t qpos = p.q_pos0 + qrow;

    // Q^T fragments (B operand): query column `col`, dims 16 s + 8 half .. +8
    // for K slice s (the K fragments use the same dim mapping).
    bf16x8 qf[8];
    {
        const uint16_t* src = p.q + b * p.qs0 + qrow * p.qs1 + h * p.qs2 + half * 8;
#pragma unroll
        for (int sl = 0; sl < 8; ++sl)
            qf[sl] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(src + 16 * sl));
    }

    // Visible key range for this workgroup (positions): up to the end of the
    // last query's chunk.
    const int64_t wg_first_q = (int64_t)qt * BQ;
    int64_t wg_last_q = wg_first_q + BQ - 1;
    wg_last_q = wg_last_q < p.Lq - 1 ? wg_last_q : p.Lq - 1;
    const int64_t r_first = p.q_pos0 + wg_first_q, r_last = p.q_pos0 + wg_last_q;
    int64_t pos_end = p.kv_len + p.cur_len;
    if (p.chunk > 0) {
        const int64_t lim = (r_last / p.chunk + 1) * p.chunk;
        pos_end = pos_end < lim ? pos_end : lim;
    }
    const int64_t cache_end = p.kv_len < pos_end ? p.kv_len : pos_end;
    const int64_t tail_end = pos_end - p.kv_len;  // tail keys visited (may be <= 0)
    const int n_cache = (int)((cache_end + BKV - 1) / BKV);
    const int n_tail = tail_end > 0 ? (int)((tail_end + BKV - 1) / BKV) : 0;
    const int n_all = n_cache + n_tail;
    // This split's share of the tile list [t_begin, t_end).
    const int t_begin = (int)((int64_t)n_all * split / p.splits);
    const int t_end = (int)((int64_t)n_all * (split + 1) / p.splits);
    // Visibility limits (exclusive key positions): this lane's query, and the
    // workgroup's first query (every key below it is visible to all lanes).
    const int64_t no_limit = p.kv_len + p.cur_len;
    const int64_t key_limit = p.chunk > 0 ? (qpos / p.chunk + 1) * p.chunk : no_limit;
    const int64_t wg_key_limit = p.chunk > 0 ? (r_first / p.chunk + 1) * p.chunk : no_limit;

    f32x16 o[4];  // O^T: [dim block], column = this lane's query
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[i][v] = 0.0f;
    Run run{-INFINITY, 0.0f, 0.0f};  // shared by the lane pair (but l)
    const float c = p.scale_log2;

    // Tile t: segment, first key index within it, key count;
    // `full`: every key exists and is visible to every query of the workgroup;
    // `lim`: keys j < lim of the tile are visible to this lane's query.
    struct Geom {
        bool cache;
        int64_t first;
        int count;
        bool full;
        int64_t pos0;  // position of the tile's key 0
    };
    auto geom = [&](int t) {
        Geom g;
        int64_t count, pos0;
        if (t < n_cache) {
            g.cache = true;
            g.first = (int64_t)t * BKV;
            count = cache_end - g.first;
            pos0 = g.first;
        } else {
            g.cache = false;
            g.first = (int64_t)(t - n_cache) * BKV;
            count = tail_end - g.first;
            pos0 = p.kv_len + g.first;
        }
        g.count = (int)(count < BKV ? count : BKV);
        g.full = g.count == BKV && pos0 + BKV <= wg_key_limit;
        g.pos0 = pos0;
        return g;
    };
    // Keys j < lim_of(g) of tile g are visible to this lane's query (taken only
    // on the masked path).
    auto lim_of = [&](const Geom& g) {
        int64_t lim64 = key_limit - g.pos0;
        lim64 = lim64 < g.count ? lim64 : g.count;
        return lim64 < 0 ? 0 : (int)lim64;
    };
    // Masks block kb of tile g, whose validity word is mw, where something is to
    // mask; mx: the block's unmasked max. Without chunks a limit is the same
    // for every query, so it joins the word.
    auto mask_block = [&](f32x16& u, int kb, const Geom& g, uint64_t mw, float mx) {
        if (g.full || p.chunk == 0) {
            const uint64_t all = g.count >= BKV ? ALL_KEYS : (1ull << g.count) - 1;
            const uint32_t w = (uint32_t)((mw & all) >> (32 * kb));
            return w == ~0u ? mx : mask_word(u, w);
        }
        return mask_raw(u, kb, half, lim_of(g), mw);
    };
    // This lane's K row (block 0) at dims 8 half .., and its V^T row (dim
    // block 0) at column unit `half` (slice 0).
    const uint32_t ka_off = col * KROW + 16 * half;
    const uint32_t va_off = K_BYTES + col * VTROW + 16 * half;
    CacheRegs<NW> regs;
    regs.s = 0.0f;
    const LaneOffs<NW> lo = lane_offsets<NW>(p);

    // Steady tiles: the prefix [t_begin, t_fast) of the range in which the
    // current and the next tile are full cache tiles (every key exists and is
    // visible to every query: nothing to mask) and the tiles written and
    // fetched are cache tiles -- the bulk of any long range. They run a loop
    // with no per-tile geometry, tail or mask branches, loading through
    // descriptors that span the (b, h) cache rows [0, cache_end) at the
    // tile's byte offset (so the span must fit 31 bits). The MASK
    // instantiations run it too: a tile's validity word then masks its blocks
    // (mask_word). The tiles up to the tail take the general loop in both
    // instantiations, the tail's tiles a loop of their own where tail_span holds.
    const int64_t full_end = cache_end < wg_key_limit ? cache_end : wg_key_limit;
    const int n_full = full_end > 0 ? (int)(full_end / BKV) : 0;
    const bool span_ok = cache_end > 0 && p.cs1 > 0 && p.ss1 > 0 &&
                         (cache_end - 1) * p.cs1 + D < ((int64_t)1 << 31) &&
                         ((cache_end - 1) * p.ss1 + 1) * 4 < ((int64_t)1 << 31);
    int t_fast = t_begin;
    if (span_ok) {
        int tf = n_full - 1;
        tf = tf < t_end - NS ? tf : t_end - NS;
        tf = tf < n_cache - NS ? tf : n_cache - NS;
        t_fast = tf > t_begin ? tf : t_begin;
    }
    const TileBase span = tile_base(p, b, h, 0, span_ok ? (int)cache_end : 0);
    const uint32_t tile_co = (uint32_t)(BKV * p.cs1), tile_so = (uint32_t)(BKV * p.ss1 * 4);

    // Software pipeline over half tiles. Tile t (u = t - t_begin) is in
    // stage u % NS; during it the wave writes tile t + NS - 1 (dequantized from
    // the prefetch registers, scales from buffer (u + NS - 1) % 2) to stage
    // (u + NS - 1) % NS and fetches the codes and scales of tile t + NS:
    //   half 0: rebase; S(t, kb 1) || probs(kb 0)
    //           PV(t, kb 0) || max(kb 1), K of t + NS - 1 written; K codes +
    //           scales of t + NS fetched
    //   half 1: rebase; S(t + 1, kb 0) || probs(kb 1)
    //           PV(t, kb 1) || max(t + 1, kb 0), V^T of t + NS - 1 written;
    //           scales of t + NS to buffer (u + NS) % 2, V codes fetched
    // NS = 2 (the loop below, written for it): K of t + 1 is written in half
    // 0 and read by S(t + 1) in half 1, so a barrier ends half 0 as well as
    // the tile. NS = 3 (the loops after it): every tile a half
    // reads was written before the barrier that ended an earlier tile, and
    // the stage written during tile t (that of t - 1) was last read in half 1
    // of t - 1, before the barrier ending it; one barrier per tile.
    // Scale buffer (u + NS) % 2 last served the write of tile t + NS - 2,
    // during tile t - 2 (NS = 3) or t - 1 (NS = 2), before a barrier.
    // The tail's tiles, from n_cache on, run a loop of their own. With the general
    // loop's geometry, per-lane addresses, unused cache writes and tail writes
    // after the steps (and, with two stages, loads waited for on the spot), a tail
    // tile took up to twice a steady cache tile's time; in its own loop it takes
    // less than one (no dequantization). 11 056 queries over 11 056 cached and
    // 11 056 tail keys with masks, in the block: 6.09 -> 5.38 ms for the whole
    // block with the 8-wave loop; the 4-wave launch of its last 304 rows per head
    // 228 -> 156 us.
    const bool tail_span = tail_end > 0 && p.us1 > 0 && ((tail_end - 1) * p.us1 + D) * 2 < ((int64_t)1 << 31);
    // Tiles below t_full exist whole and are visible to every query.
    const int64_t tail_vis = wg_key_limit - p.kv_len, tail_full = tail_end < tail_vis ? tail_end : tail_vis;
    const int t_full = n_cache + (tail_full > 0 ? (int)(tail_full / BKV) : 0);
    // Descriptors spanning the tail rows of (b, h), and tile t's byte offset.
    auto tail_rsrc = [&](const uint16_t* base) {
        return tile_rsrc(base + b * p.us0 + h * p.us2, ((tail_end - 1) * p.us1 + D) * 2);
    };
    auto tail_off = [&](int t) { return (uint32_t)((int64_t)(t - n_cache) * BKV * p.us1 * 2); };
    if constexpr (NS == 2) {
        if (t_end > t_begin) {
            f32x16 sa, sb;
            float mxa, mxb;
            uint64_t mw;  // validity word of tile t
            Geom g = geom(t_begin);
            {
                if (g.cache) {
                    const TileBase tb = tile_base(p, b, h, g.first, g.count);
                    load_k<NW, MASK>(lo, regs, tb, g.count);
                    load_v<NW>(lo, regs, tb);
                    __builtin_amdgcn_s_waitcnt(0);
                    if (threadIdx.x < 2 * BKV) sbuf[threadIdx.x] = regs.s;
                    __syncthreads();
                    store_tile<FMT, NW, MASK>(regs, smem, sbuf);
                } else {
                    copy_tail_k<NW, MASK>(p, b, h, g.first, g.count, smem);
                    copy_tail_v<NW>(p, b, h, g.first, g.count, smem);
                }
                if (t_begin + 1 < t_end) {
                    const Geom g1 = geom(t_begin + 1);
                    if (g1.cache) {
                        const TileBase tb = tile_base(p, b, h, g1.first, g1.count);
                        load_k<NW, MASK>(lo, regs, tb, g1.count);
                        load_v<NW>(lo, regs, tb);
                    }
                }
                // Everything issued so far (the Q fragments included) has landed;
                // inside the loop the only loads in flight are the prefetch.
                __builtin_amdgcn_s_waitcnt(0);
                if (threadIdx.x < 2 * BKV) sbuf[SB_FLOATS + threadIdx.x] = regs.s;
                __syncthreads();
                mw = tile_mask<MASK>(smem);
                sa = s_block(smem + ka_off, qf);
                mxa = raw_max(sa);
                if (!g.full || mw != ALL_KEYS) mxa = mask_block(sa, 0, g, mw, mxa);
            }
            int t = t_begin;
            {
                // steady tiles (see t_fast): fetch tile t + 2 at offsets fco / fso.
                // With validity masks (MASK) each tile's word travels with its
                // K write; a tile whose word is not all ones masks its blocks.
                uint32_t fco = (uint32_t)((int64_t)(t + 2) * BKV * p.cs1);
                uint32_t fso = (uint32_t)((int64_t)(t + 2) * BKV * p.ss1 * 4);
                for (; t < t_fast; ++t) {
                    const int u = t - t_begin;
                    const uint8_t* st = smem + (u & 1) * STAGE;
                    uint8_t* nst = smem + ((u & 1) ^ 1) * STAGE;
                    const float* nsb = sbuf + ((u & 1) ^ 1) * SB_FLOATS;
                    f16x8 pf[2];
                    rebase(mxa, c, run, o);
                    sb = step_a(sa, c, run.nm, run.l, pf, st + ka_off + 32 * KROW, qf);
                    mxb = step_b<FMT, NW, 1>(pf, st + va_off, 0, o, sb, regs, nst, nsb);
                    if constexpr (MASK) {
                        store_mask<NW, MASK>(regs, nst);
                        if ((uint32_t)(mw >> 32) != ~0u) mxb = mask_word(sb, (uint32_t)(mw >> 32));
                    }
                    load_k<NW, MASK>(lo, regs, span, BKV, fco, fso, (int64_t)(t + 2) * BKV);
                    __syncthreads();
                    rebase(mxb, c, run, o);
                    sa = step_a(sb, c, run.nm, run.l, pf, nst + ka_off, qf);
                    mxa = step_b<FMT, NW, 2>(pf, st + va_off, 1, o, sa, regs, nst, nsb);
                    if constexpr (MASK) {
                        mw = tile_mask<MASK>(nst);  // tile t + 1
                        if ((uint32_t)mw != ~0u) mxa = mask_word(sa, (uint32_t)mw);
                    }
                    if (threadIdx.x < 2 * BKV) sbuf[(u & 1) * SB_FLOATS + threadIdx.x] = regs.s;
                    load_v<NW>(lo, regs, span, fco);
                    __syncthreads();
                    fco += tile_co;
                    fso += tile_so;
                }
                if (t > t_begin) g = geom(t);
            }
            const int t_tail = tail_span && t_end > n_cache ? (t > n_cache ? t : n_cache) : t_end;
            for (; t < t_tail; ++t) {
                const int u = t - t_begin;
                const uint8_t* st = smem + (u & 1) * STAGE;
                uint8_t* nst = smem + ((u & 1) ^ 1) * STAGE;
                const float* nsb = sbuf + ((u & 1) ^ 1) * SB_FLOATS;  // scales of tile t + 1
                const bool has_next = t + 1 < t_end;
                const Geom gn = geom(has_next ? t + 1 : t);
                const bool fetch2 = t + 2 < t_end;
                const Geom g2 = geom(fetch2 ? t + 2 : t);
                f16x8 pf[2];

                // ---- half 0
                rebase(mxa, c, run, o);
                sb = step_a(sa, c, run.nm, run.l, pf, st + ka_off + 32 * KROW, qf);
                // K (and validity word) of tile t + 1 from the prefetch registers
                // (a tail tile or the end of the range is handled right after:
                // the stage is not read before the barrier).
                mxb = step_b<FMT, NW, 1>(pf, st + va_off, 0, o, sb, regs, nst, nsb);
                store_mask<NW, MASK>(regs, nst);
                if (!g.full || mw != ALL_KEYS) mxb = mask_block(sb, 1, g, mw, mxb);
                if (has_next && !gn.cache) copy_tail_k<NW, MASK>(p, b, h, gn.first, gn.count, nst);
                const int n2 = fetch2 && g2.cache ? g2.count : 0;  // 0: no fetch (zeros)
                load_k<NW, MASK>(lo, regs, tile_base(p, b, h, g2.first, n2), n2);
                __syncthreads();

                // ---- half 1 (on the last tile the S block of "tile t + 1" reads
                // stale LDS; its result is never used)
                const uint64_t mwn = tile_mask<MASK>(nst);
                rebase(mxb, c, run, o);
                sa = step_a(sb, c, run.nm, run.l, pf, nst + ka_off, qf);
                mxa = step_b<FMT, NW, 2>(pf, st + va_off, 1, o, sa, regs, nst, nsb);
                if (!gn.full || mwn != ALL_KEYS) mxa = mask_block(sa, 0, gn, mwn, mxa);
                if (has_next && !gn.cache) copy_tail_v<NW>(p, b, h, gn.first, gn.count, nst);
                // (without a fetch: zeros into a scale buffer no write reads)
                if (threadIdx.x < 2 * BKV) sbuf[(u & 1) * SB_FLOATS + threadIdx.x] = regs.s;
                load_v<NW>(lo, regs, tile_base(p, b, h, g2.first, n2));
                __syncthreads();
                g = gn;
                mw = mwn;
            }
            if (t < t_end) {
                const __amdgpu_buffer_rsrc_t tk = tail_rsrc(p.kcur), tv = tail_rsrc(p.vcur);
                const TailOffs<NW> to = tail_offsets<NW>(p);
                TailRegs<NW> tregs;  // tile t + 1 (past the end: zeros that no tile reads)
                load_tail_span_k<NW, MASK>(p, b, to, tk, tail_off(t + 1), (int64_t)(t + 1 - n_cache) * BKV, tail_end,
                                           tregs);
                load_tail_span_v<NW>(to, tv, tail_off(t + 1), tregs);
                uint32_t co = tail_off(t + 2);
                const uint32_t dco = (uint32_t)(BKV * p.us1 * 2);
                for (; t < t_end; ++t) {
                    const int u = t - t_begin;
                    const uint8_t* st = smem + (u & 1) * STAGE;
                    uint8_t* nst = smem + ((u & 1) ^ 1) * STAGE;
                    f16x8 pf[2];
                    rebase(mxa, c, run, o);
                    sb = step_a(sa, c, run.nm, run.l, pf, st + ka_off + 32 * KROW, qf);
                    mxb = step_b_with(pf, st + va_off, 0, o, sb, [&](int i) __attribute__((always_inline)) {
                        if (i & 1) store_tail_k_part<NW>(tregs, nst, i >> 2, (i >> 1) & 1);
                    });
                    store_tail_mask<NW, MASK>(tregs, nst);
                    if (t >= t_full || mw != ALL_KEYS) mxb = mask_block(sb, 1, geom(t), mw, mxb);
                    load_tail_span_k<NW, MASK>(p, b, to, tk, co, (int64_t)(t + 2 - n_cache) * BKV, tail_end, tregs);
                    __syncthreads();
                    const uint64_t mwn = tile_mask<MASK>(nst);
                    rebase(mxb, c, run, o);
                    sa = step_a(sb, c, run.nm, run.l, pf, nst + ka_off, qf);
                    mxa = step_b_with(pf, st + va_off, 1, o, sa, [&](int i) __attribute__((always_inline)) {
                        store_tail_v_part<NW>(tregs, nst, i);
                    });
                    if (t + 1 >= t_full || mwn != ALL_KEYS)  // (unused on the last tile)
                        mxa = mask_block(sa, 0, geom(t + 1 < t_end ? t + 1 : t), mwn, mxa);
                    load_tail_span_v<NW>(to, tv, co, tregs);
                    __syncthreads();
                    co += dco;
                    mw = mwn;
                }
            }
        }
    } else {
        if (t_end > t_begin) {
            f32x16 sa, sb;
            float mxa, mxb;
            // Prologue: tiles t_begin .. t_begin + NS - 2 written, the codes of
            // t_begin + NS - 1 in the prefetch registers with their scales in
            // buffer (NS - 1) % 2. Tiles k < NS - 1: load, scales to buffer k % 2,
            // barrier, dequantizing write to stage k (buffer k % 2 is rewritten
            // only after the next barrier, which follows this write).
#pragma unroll
            for (int k = 0; k < NS - 1; ++k) {
                const int t = t_begin + k;
                if (t >= t_end) break;
                const Geom gk = geom(t);
                if (gk.cache) {
                    const TileBase tb = tile_base(p, b, h, gk.first, gk.count);
                    load_k<NW, MASK>(lo, regs, tb, gk.count);
                    load_v<NW>(lo, regs, tb);
                    __builtin_amdgcn_s_waitcnt(0);
                    if (threadIdx.x < 2 * BKV) sbuf[(k & 1) * SB_FLOATS + threadIdx.x] = regs.s;
                    __syncthreads();
                    store_tile<FMT, NW, MASK>(regs, smem + k * STAGE, sbuf + (k & 1) * SB_FLOATS);
                } else {
                    copy_tail_k<NW, MASK>(p, b, h, gk.first, gk.count, smem + k * STAGE);
                    copy_tail_v<NW>(p, b, h, gk.first, gk.count, smem + k * STAGE);
                }
            }
            TailRegs<NW> tregs;  // a tail tile's bf16 K/V, loaded one tile ahead of its write
            if (t_begin + NS - 1 < t_end) {
                const Geom gk = geom(t_begin + NS - 1);
                if (gk.cache) {
                    const TileBase tb = tile_base(p, b, h, gk.first, gk.count);
                    load_k<NW, MASK>(lo, regs, tb, gk.count);
                    load_v<NW>(lo, regs, tb);
                } else {
                    load_tail_k<NW, MASK>(p, b, h, gk.first, gk.count, tregs);
                    load_tail_v<NW>(p, b, h, gk.first, gk.count, tregs);
                }
            }
            // Everything issued so far (the Q fragments included) has landed;
            // inside the loop the only loads in flight are the prefetch.
            __builtin_amdgcn_s_waitcnt(0);
            if (threadIdx.x < 2 * BKV) sbuf[((NS - 1) & 1) * SB_FLOATS + threadIdx.x] = regs.s;
            __syncthreads();
            Geom g = geom(t_begin);
            uint64_t mw = tile_mask<MASK>(smem);  // validity word of tile t
            sa = s_block(smem + ka_off, qf);
            mxa = raw_max(sa);
                if (!g.full || mw != ALL_KEYS) mxa = mask_block(sa, 0, g, mw, mxa);
            int t = t_begin;
            {
                // steady tiles (see t_fast): fetch tile t + NS at offsets fco / fso
                // (validity words as in the two-stage loop above)
                uint32_t fco = (uint32_t)((int64_t)(t + NS) * BKV * p.cs1);
                uint32_t fso = (uint32_t)((int64_t)(t + NS) * BKV * p.ss1 * 4);
                int s0 = 0;  // stage of tile t, (t - t_begin) % NS
                for (; t < t_fast; ++t) {
                    const int u = t - t_begin;
                    const int s1 = s0 == NS - 1 ? 0 : s0 + 1;  // tile t + 1
                    const int sw = s0 == 0 ? NS - 1 : s0 - 1;  // tile t + NS - 1
                    const uint8_t* st = smem + s0 * STAGE;
                    const uint8_t* st1 = smem + s1 * STAGE;
                    uint8_t* wst = smem + sw * STAGE;
                    const float* wsb = sbuf + ((u + NS - 1) & 1) * SB_FLOATS;
                    f16x8 pf[2];
                    const uint64_t mwn = tile_mask<MASK>(st1);  // tile t + 1
                    rebase(mxa, c, run, o);
                    sb = step_a(sa, c, run.nm, run.l, pf, st + ka_off + 32 * KROW, qf);
                    mxb = step_b<FMT, NW, 1>(pf, st + va_off, 0, o, sb, regs, wst, wsb);
                    if constexpr (MASK) {
                        store_mask<NW, MASK>(regs, wst);
                        if ((uint32_t)(mw >> 32) != ~0u) mxb = mask_word(sb, (uint32_t)(mw >> 32));
                    }
                    load_k<NW, MASK>(lo, regs, span, BKV, fco, fso, (int64_t)(t + NS) * BKV);
                    rebase(mxb, c, run, o);
                    sa = step_a(sb, c, run.nm, run.l, pf, st1 + ka_off, qf);
                    mxa = step_b<FMT, NW, 2>(pf, st + va_off, 1, o, sa, regs, wst, wsb);
                    if constexpr (MASK) {
                        if ((uint32_t)mwn != ~0u) mxa = mask_word(sa, (uint32_t)mwn);
                        mw = mwn;
                    }
                    if (threadIdx.x < 2 * BKV) sbuf[((u + NS) & 1) * SB_FLOATS + threadIdx.x] = regs.s;
                    load_v<NW>(lo, regs, span, fco);
                    __syncthreads();
                    fco += tile_co;
                    fso += tile_so;
                    s0 = s1;
                }
                if (t > t_begin) g = geom(t);
            }
            const int t_tail = tail_span && t_end > n_cache ? (t > n_cache ? t : n_cache) : t_end;
            for (; t < t_tail; ++t) {
                const int u = t - t_begin;
                const uint8_t* st = smem + (u % NS) * STAGE;              // tile t
                const uint8_t* st1 = smem + ((u + 1) % NS) * STAGE;       // tile t + 1
                uint8_t* wst = smem + ((u + NS - 1) % NS) * STAGE;        // tile t + NS - 1
                const float* wsb = sbuf + ((u + NS - 1) & 1) * SB_FLOATS; // its scales
                const bool has_next = t + 1 < t_end;
                const Geom gn = geom(has_next ? t + 1 : t);
                const bool write = t + NS - 1 < t_end;
                const Geom gw = geom(write ? t + NS - 1 : t);
                const bool fetch = t + NS < t_end;
                const Geom gf = geom(fetch ? t + NS : t);
                f16x8 pf[2];
                const uint64_t mwn = tile_mask<MASK>(st1);  // tile t + 1 (stale on the last tile)

                // ---- half 0
                rebase(mxa, c, run, o);
                sb = step_a(sa, c, run.nm, run.l, pf, st + ka_off + 32 * KROW, qf);
                // K (and validity word) of tile t + NS - 1 from the prefetch
                // registers (a tail tile or the end of the range is handled
                // right after: the stage is not read before the barrier).
                mxb = step_b<FMT, NW, 1>(pf, st + va_off, 0, o, sb, regs, wst, wsb);
                store_mask<NW, MASK>(regs, wst);
                if (!g.full || mw != ALL_KEYS) mxb = mask_block(sb, 1, g, mw, mxb);
                if (write && !gw.cache) store_tail_k<NW, MASK>(tregs, wst);
                const int nf = fetch && gf.cache ? gf.count : 0;  // 0: no fetch (zeros)
                load_k<NW, MASK>(lo, regs, tile_base(p, b, h, gf.first, nf), nf);
                if (fetch && !gf.cache) load_tail_k<NW, MASK>(p, b, h, gf.first, gf.count, tregs);

                // ---- half 1 (on the last tile the S block of "tile t + 1" reads
                // stale LDS; its result is never used)
                rebase(mxb, c, run, o);
                sa = step_a(sb, c, run.nm, run.l, pf, st1 + ka_off, qf);
                mxa = step_b<FMT, NW, 2>(pf, st + va_off, 1, o, sa, regs, wst, wsb);
                if (!gn.full || mwn != ALL_KEYS) mxa = mask_block(sa, 0, gn, mwn, mxa);
                if (write && !gw.cache) store_tail_v<NW>(tregs, wst);
                // (without a fetch: zeros into a scale buffer no write reads)
                if (threadIdx.x < 2 * BKV) sbuf[((u + NS) & 1) * SB_FLOATS + threadIdx.x] = regs.s;
                load_v<NW>(lo, regs, tile_base(p, b, h, gf.first, nf));
                if (fetch && !gf.cache) load_tail_v<NW>(p, b, h, gf.first, gf.count, tregs);
                __syncthreads();
                g = gn;
                mw = mwn;
            }
            if (t < t_end) {
                const __amdgpu_buffer_rsrc_t tk = tail_rsrc(p.kcur), tv = tail_rsrc(p.vcur);
                const TailOffs<NW> to = tail_offsets<NW>(p);
                uint32_t co = tail_off(t + NS);
                const uint32_t dco = (uint32_t)(BKV * p.us1 * 2);
                int s0 = (t - t_begin) % NS;
                for (; t < t_end; ++t) {
                    const int s1 = s0 == NS - 1 ? 0 : s0 + 1, sw = s0 == 0 ? NS - 1 : s0 - 1;
                    const uint8_t* st = smem + s0 * STAGE;
                    const uint8_t* st1 = smem + s1 * STAGE;
                    uint8_t* wst = smem + sw * STAGE;
                    f16x8 pf[2];
                    const uint64_t mwn = tile_mask<MASK>(st1);
                    rebase(mxa, c, run, o);
                    sb = step_a(sa, c, run.nm, run.l, pf, st + ka_off + 32 * KROW, qf);
                    mxb = step_b_with(pf, st + va_off, 0, o, sb, [&](int i) __attribute__((always_inline)) {
                        if (i == 3 || i == 6) store_tail_k_part<NW>(tregs, wst, 0, i == 6);
                    });
                    store_tail_mask<NW, MASK>(tregs, wst);
                    if (t >= t_full || mw != ALL_KEYS) mxb = mask_block(sb, 1, geom(t), mw, mxb);
                    load_tail_span_k<NW, MASK>(p, b, to, tk, co, (int64_t)(t + NS - n_cache) * BKV, tail_end, tregs);
                    rebase(mxb, c, run, o);
                    sa = step_a(sb, c, run.nm, run.l, pf, st1 + ka_off, qf);
                    mxa = step_b_with(pf, st + va_off, 1, o, sa, [&](int i) __attribute__((always_inline)) {
                        if (i & 1) store_tail_v_part<NW>(tregs, wst, i >> 1);
                    });
                    if (t + 1 >= t_full || mwn != ALL_KEYS)  // (unused on the last tile)
                        mxa = mask_block(sa, 0, geom(t + 1 < t_end ? t + 1 : t), mwn, mxa);
                    load_tail_span_v<NW>(to, tv, co, tregs);
                    __syncthreads();
                    co += dco;
                    s0 = s1;
                    mw = mwn;
                }
            }
        }
    }
    const float l = run.l + __shfl_xor(run.l, 32, 64);
    const float m = run.m;

    // ---- epilogue: O = O^T / l; the lane holds dims 32 db + 8 (v/4) + 4 half + v%4
    if (p.splits > 1) {
        // Unnormalized partial result of this key range, merged by attn_combine_kernel.
        if (qvalid) {
            const int64_t qi = ((((int64_t)split * (p.work / p.splits / p.q_tiles / p.H)) + b) * p.H + h) * p.Lq + row;
            float* dst = p.ws_o + qi * D;
#pragma unroll
            for (int db = 0; db < 4; ++db)
#pragma unroll
                for (int vq = 0; vq < 4; ++vq) {
                    const int d = db * 32 + vq * 8 + half * 4;
                    *reinterpret_cast<float4*>(dst + d) =
                        make_float4(o[db][vq * 4], o[db][vq * 4 + 1], o[db][vq * 4 + 2], o[db][vq * 4 + 3]);
                }
            if (half == 0) *reinterpret_cast<float2*>(p.ws_ml + qi * 2) = make_float2(m, l);
        }
        return;
    }
    if (qvalid) {
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
        uint16_t* dst = p.out + b * p.os0 + row * p.os1 + h * p.os2;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int vq = 0; vq < 4; ++vq) {
                const int d = db * 32 + vq * 8 + half * 4;
                const uint32_t w0 = f32_to_bf16_bits(o[db][vq * 4] * inv) |
                                    (f32_to_bf16_bits(o[db][vq * 4 + 1] * inv) << 16);
                const uint32_t w1 = f32_to_bf16_bits(o[db][vq * 4 + 2] * inv) |
                                    (f32_to_bf16_bits(o[db][vq * 4 + 3] * inv) << 16);
                *reinterpret_cast<uint2*>(dst + d) = make_uint2(w0, w1);
            }
    }
}

// Merge of the per-split partial results: with M = max_s m_s,
// O = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s (0 when no key was visible).
// 8 (batch, head, query) rows per 256-thread block, 32 threads per row, each
// owning 4 consecutive dimensions: 16-byte loads of the partials and one
// 8-byte store. Every element is the same chain of operations in split order
// as with one thread per dimension, so the result does not depend on the
// block shape.
constexpr int COMBINE_ROWS = 8;
__global__ __launch_bounds__(256) void attn_combine_kernel(const float* __restrict__ ws_o,
                                                           const float* __restrict__ ws_ml,
                                                           int splits, int64_t rows_per_split,
                                                           int64_t Lq, int64_t H, uint16_t* out,
                                                           int64_t os0, int64_t os1, int64_t os2) {
    const int64_t r = (int64_t)blockIdx.x * COMBINE_ROWS + (threadIdx.x >> 5);  // (b * H + h) * Lq + q
    if (r >= rows_per_split) return;
    const int d = (threadIdx.x & 31) * 4;
    float M = -INFINITY;
    for (int sp = 0; sp < splits; ++sp) M = fmaxf(M, ws_ml[(sp * rows_per_split + r) * 2]);
    const float Muse = M == -INFINITY ? 0.0f : M;
    float den = 0.0f;
    float num[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int sp = 0; sp < splits; ++sp) {
        const int64_t idx = sp * rows_per_split + r;
        const float2 ml = *reinterpret_cast<const float2*>(ws_ml + idx * 2);
        const float4 ov = *reinterpret_cast<const float4*>(ws_o + idx * D + d);
        const float wgt = __builtin_amdgcn_exp2f(ml.x - Muse);
        den = fmaf(wgt, ml.y, den);
        num[0] = fmaf(wgt, ov.x, num[0]);
        num[1] = fmaf(wgt, ov.y, num[1]);
        num[2] = fmaf(wgt, ov.z, num[2]);
        num[3] = fmaf(wgt, ov.w, num[3]);
    }
    const int64_t q = r % Lq, h = (r / Lq) % H, b = r / (Lq * H);
    uint32_t o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = f32_to_bf16_bits(den > 0.0f ? num[e] / den : 0.0f);
    *reinterpret_cast<uint2*>(out + b * os0 + q * os1 + h * os2 + d) =
        make_uint2(o[0] | (o[1] << 16), o[2] | (o[3] << 16));
}

}  // namespace attn
}  // namespace hn

using namespace hn;

// Split selection for the 4-wave kernel: a launch wants at least two
// workgroups per CU (two fit per CU by LDS and registers). When (batch x heads
// x query tiles) falls short, the key range of each query tile is split so
// that the grid fills the device (the decode-style case: a few hundred
// queries over a long cache); each split keeps at least 16 key tiles.
static int attn_splits(int64_t B, int64_t Lq, int64_t H, int64_t kv_len, int64_t cur_len, int cus) {
    const int64_t work = B * H * ((Lq + attn::Shape<4>::BQ - 1) / attn::Shape<4>::BQ);
    const int64_t target = 2LL * cus;
    if (work <= 0 || work >= target) return 1;
    const int64_t tiles = (kv_len + cur_len + attn::BKV - 1) / attn::BKV;
    // Round down: the kernel holds two workgroups per CU, so work * sp <= target
    // keeps the whole launch in one round (one more workgroup would need a second).
    int64_t sp = target / work;
    const int64_t cap = tiles / 16;
    if (sp > cap) sp = cap;
    return sp > 1 ? (int)sp : 1;
}

// Launch plan: query rows [0, rows8) go to the 8-wave kernel (whole 256-query
// tiles, no key split), rows [rows8, Lq) to the 4-wave kernel with `splits`
// key-range splits.
//
// Model, in units of one full round of 4-wave workgroups (2 per CU, 128
// queries each, which takes as long per key tile as one round of 8-wave
// workgroups, 1 per CU, 256 queries each -- the 8-wave round measures 0.92 of
// it at 86400 keys, so K8_ROUND = 0.92):
//   4-wave only: ceil(n4 / 2C) rounds, n4 = B H ceil(Lq / 128);
//   8-wave over k tiles of 256 rows per (batch, head): ceil(B H k / C)
//                K8_ROUND rounds, plus the other Lq - 256 k rows on the
//                4-wave kernel, split sp ways: ceil(nr sp / 2C) / sp rounds.
// Every k from floor(Lq / 256) down is tried, so that a few rows past a
// whole number of 8-wave rounds (a chunk's text tokens beside its 10 800
// image tokens: 43 tiles x 24 heads = 4.03 rounds, i.e. 5) go to the split
// 4-wave launch instead of a nearly empty extra round. The 8-wave kernel is
// used only when it fills every CU at least once (B H k >= C) and the model
// says it is faster: a partial last round of 1-per-CU workgroups idles half
// the SIMD slots a 4-wave round would keep busy.
struct AttnPlan {
    int64_t rows8;
    int splits;
};

static AttnPlan attn_plan(int64_t B, int64_t Lq, int64_t H, int64_t kv_len, int64_t cur_len) {
    constexpr double K8_ROUND = 0.92;
    const int cus = device_cus();
    AttnPlan plan{0, 1};
    const int64_t bh = B * H;
    const int64_t n4 = bh * ((Lq + attn::Shape<4>::BQ - 1) / attn::Shape<4>::BQ);
    double best = (double)((n4 + 2 * cus - 1) / (2 * cus));
    for (int64_t k = Lq / attn::Shape<8>::BQ; k > 0 && bh * k >= cus; --k) {
        const int64_t n8 = bh * k;
        double r8 = K8_ROUND * (double)((n8 + cus - 1) / cus);
        const int64_t rows8 = k * attn::Shape<8>::BQ;
        const int64_t rest = Lq - rows8;
        if (rest > 0) {
            const int sp = attn_splits(B, rest, H, kv_len, cur_len, cus);
            const int64_t nr = bh * ((rest + attn::Shape<4>::BQ - 1) / attn::Shape<4>::BQ) * sp;
            r8 += (double)((nr + 2 * cus - 1) / (2 * cus)) / sp;
        }
        if (r8 < best) {
            best = r8;
            plan.rows8 = rows8;
        }
        if (r8 > best + 1.0) break;  // fewer tiles only add 4-wave rounds from here
    }
    plan.splits = attn_splits(B, Lq - plan.rows8, H, kv_len, cur_len, cus);
    return plan;
}

static int64_t plan_workspace(const AttnPlan& plan, int64_t B, int64_t Lq, int64_t H) {
    if (plan.splits <= 1) return 0;
    return (int64_t)plan.splits * B * H * (Lq - plan.rows8) * (attn::D + 2) * (int64_t)sizeof(float);
}

extern "C" int64_t hn_attn_fp8kv_workspace_size(int64_t B, int64_t Lq, int64_t H, int64_t D,
                                                int64_t kv_len, int64_t cur_len) {
    if (B <= 0 || Lq <= 0 || H <= 0 || D != attn::D || kv_len < 0 || cur_len < 0) return 0;
    return plan_workspace(attn_plan(B, Lq, H, kv_len, cur_len), B, Lq, H);
}

// The kernel instantiation for the format, with or without key-validity masks.
template <int NW, bool MASK>
static void launch_kernel(const attn::Params& p, dim3 grid, hipStream_t stream) {
    if (p.fmt == HN_KV_FP8)
        attn::attn_fp8kv_kernel<HN_KV_FP8, NW, MASK><<<grid, attn::Shape<NW>::NT, 0, stream>>>(p);
    else
        attn::attn_fp8kv_kernel<HN_KV_INT8, NW, MASK><<<grid, attn::Shape<NW>::NT, 0, stream>>>(p);
}


// One launch of the NW-wave kernel over query rows [row0, row0 + rows) of p's
// problem (p.Lq = all rows), with `sp` key-range splits merged through the
// workspace by attn_combine_kernel.
template <int NW>
static int launch_rows(attn::Params p, int64_t B, int64_t row0, int64_t rows, int sp, void* workspace,
                       hipStream_t stream) {
    constexpr int BQ = attn::Shape<NW>::BQ;
    p.q += row0 * p.qs1;
    p.out += row0 * p.os1;
    p.q_pos0 += row0;
    p.Lq = rows;
    const int64_t qt = (rows + BQ - 1) / BQ;
    const int64_t work = B * p.H * qt * sp;
    HN_REQUIRE(work <= 0x3fffffffLL, HN_E_ARG, "hn_attn_fp8kv: too much work for one launch");
    p.q_tiles = (int)qt;
    p.splits = sp;
    p.work = (int)work;
    p.per_xcd = (int)((work + 7) / 8);
    p.ws_o = sp > 1 ? (float*)workspace : nullptr;
    p.ws_ml = sp > 1 ? (float*)workspace + (int64_t)sp * B * p.H * rows * attn::D : nullptr;
    const dim3 grid((unsigned)(8 * (int64_t)p.per_xcd));
    if (p.kvalid || p.uvalid) launch_kernel<NW, true>(p, grid, stream);
    else launch_kernel<NW, false>(p, grid, stream);
    int rc = check_launch("hn_attn_fp8kv");
    if (rc != HN_OK || sp <= 1) return rc;
    const int64_t nrows = B * p.H * rows;
    HN_REQUIRE(nrows <= 0x7fffffffLL, HN_E_ARG, "hn_attn_fp8kv: too many rows to combine");
    attn::attn_combine_kernel<<<(unsigned)((nrows + attn::COMBINE_ROWS - 1) / attn::COMBINE_ROWS), 256, 0, stream>>>(
        p.ws_o, p.ws_ml, sp, nrows, rows, p.H, p.out, p.os0, p.os1, p.os2);
    return check_launch("hn_attn_fp8kv (combine)");
}

// Argument checks and parameter block shared by the attention entry points.
// Returns HN_OK with *pp and *plan filled, or an error code (nothing enqueued).
static int attn_setup(int fmt, const void* q, const int64_t* qs, int64_t B, int64_t Lq, int64_t H,
                      int64_t D, const void* kc, const void* vc, const int64_t* cs, const float* ks,
                      const float* vs, const int64_t* ss, int64_t cache_cap, int64_t kv_len,
                      const uint8_t* cache_valid, int64_t cvs, const void* kcur, const void* vcur,
                      const int64_t* curs, int64_t cur_len, const uint8_t* cur_valid, int64_t uvs,
                      int64_t q_pos0, int64_t chunk_len, float softmax_scale, void* out,
                      const int64_t* os, attn::Params* pp, AttnPlan* plan, bool* empty) {
    HN_REQUIRE(fmt == HN_KV_FP8 || fmt == HN_KV_INT8, HN_E_ARG, "hn_attn_fp8kv: unknown KV format");
    HN_REQUIRE(D == attn::D, HN_E_ARG, "hn_attn_fp8kv: head dim must be 128");
    HN_REQUIRE(B >= 0 && Lq >= 0 && H > 0 && kv_len >= 0 && cur_len >= 0 && q_pos0 >= 0, HN_E_ARG,
               "hn_attn_fp8kv: invalid shape");
    HN_REQUIRE(kv_len <= cache_cap, HN_E_ARG, "hn_attn_fp8kv: kv_len exceeds the cache capacity");
    HN_REQUIRE(softmax_scale > 0.0f && softmax_scale <= 3.4028234e38f, HN_E_ARG,
               "hn_attn_fp8kv: softmax_scale must be finite and positive");
    HN_REQUIRE(cvs >= 0 && uvs >= 0, HN_E_ARG, "hn_attn_fp8kv: negative validity stride");
    HN_REQUIRE(qs && os && (kv_len == 0 || (cs && ss)) && (cur_len == 0 || curs), HN_E_ARG,
               "hn_attn_fp8kv: null stride array");
    HN_REQUIRE(qs[3] == 1 && os[3] == 1, HN_E_ARG, "hn_attn_fp8kv: head dim must be contiguous");
    HN_REQUIRE(qs[0] % 8 == 0 && qs[1] % 8 == 0 && qs[2] % 8 == 0 && os[0] % 4 == 0 &&
                   os[1] % 4 == 0 && os[2] % 4 == 0,
               HN_E_ARG, "hn_attn_fp8kv: q/out strides misaligned");
    HN_REQUIRE(aligned(q, 16) && aligned(out, 8), HN_E_ARG, "hn_attn_fp8kv: q/out misaligned");
    if (kv_len > 0) {
        HN_REQUIRE(kc && vc && ks && vs, HN_E_ARG, "hn_attn_fp8kv: null cache pointer");
        HN_REQUIRE(cs[3] == 1 && cs[0] % 16 == 0 && cs[1] % 16 == 0 && cs[2] % 16 == 0, HN_E_ARG,
                   "hn_attn_fp8kv: cache strides must be multiples of 16 bytes");
        HN_REQUIRE(cs[0] >= 0 && cs[1] > 0 && cs[2] >= 0 && ss[0] >= 0 && ss[1] > 0 && ss[2] >= 0,
                   HN_E_ARG, "hn_attn_fp8kv: invalid cache strides");
        HN_REQUIRE(aligned(kc, 16) && aligned(vc, 16), HN_E_ARG, "hn_attn_fp8kv: cache misaligned");
    }
    if (cur_len > 0) {
        HN_REQUIRE(kcur && vcur, HN_E_ARG, "hn_attn_fp8kv: null tail pointer");
        HN_REQUIRE(curs[3] == 1 && curs[0] % 8 == 0 && curs[1] % 8 == 0 && curs[2] % 8 == 0,
                   HN_E_ARG, "hn_attn_fp8kv: tail strides must be multiples of 8");
        HN_REQUIRE(aligned(kcur, 16) && aligned(vcur, 16), HN_E_ARG, "hn_attn_fp8kv: tail misaligned");
    }
    *empty = B == 0 || Lq == 0;
    if (*empty) return HN_OK;
    HN_REQUIRE(out && q, HN_E_ARG, "hn_attn_fp8kv: null q/out");
    const int rc = require_gfx950("hn_attn_fp8kv");
    if (rc != HN_OK) return rc;
    attn::Params& p = *pp;
    p.q = (const uint16_t*)q;
    p.kc = (const uint8_t*)kc; p.vc = (const uint8_t*)vc;
    p.ks = ks; p.vs = vs;
    p.kcur = (const uint16_t*)kcur; p.vcur = (const uint16_t*)vcur;
    p.out = (uint16_t*)out;
    p.kvalid = kv_len > 0 ? cache_valid : nullptr;
    p.uvalid = cur_len > 0 ? cur_valid : nullptr;
    p.kvs = cvs; p.uvs = uvs;
    p.qs0 = qs[0]; p.qs1 = qs[1]; p.qs2 = qs[2];
    if (kv_len > 0) {
        p.cs0 = cs[0]; p.cs1 = cs[1]; p.cs2 = cs[2];
        p.ss0 = ss[0]; p.ss1 = ss[1]; p.ss2 = ss[2];
    } else {
        p.cs0 = p.cs1 = p.cs2 = p.ss0 = p.ss1 = p.ss2 = 0;
    }
    if (cur_len > 0) {
        p.us0 = curs[0]; p.us1 = curs[1]; p.us2 = curs[2];
    } else {
        p.us0 = p.us1 = p.us2 = 0;
    }
    p.os0 = os[0]; p.os1 = os[1]; p.os2 = os[2];
    p.Lq = Lq; p.H = H; p.kv_len = kv_len; p.cur_len = cur_len;
    p.q_pos0 = q_pos0; p.chunk = chunk_len;
    p.scale_log2 = softmax_scale * 1.4426950408889634f;
    p.fmt = fmt;
    *plan = attn_plan(B, Lq, H, kv_len, cur_len);
    return HN_OK;
}

static int attn_run(const attn::Params& p, const AttnPlan& plan, int64_t B, int64_t Lq, void* workspace,
                    hipStream_t st) {
    if (plan.rows8 > 0) {
        const int rc = launch_rows<8>(p, B, 0, plan.rows8, 1, nullptr, st);
        if (rc != HN_OK || plan.rows8 == Lq) return rc;
    }
    return launch_rows<4>(p, B, plan.rows8, Lq - plan.rows8, plan.splits, workspace, st);
}

extern "C" int hn_attn_fp8kv(int fmt, const void* q, const int64_t* qs, int64_t B, int64_t Lq,
                             int64_t H, int64_t D, const void* kc, const void* vc,
                             const int64_t* cs, const float* ks, const float* vs,
                             const int64_t* ss, int64_t cache_cap, int64_t kv_len,
                             const uint8_t* cache_valid, int64_t cache_valid_stride,
                             const void* kcur, const void* vcur, const int64_t* curs,
                             int64_t cur_len, const uint8_t* cur_valid, int64_t cur_valid_stride,
                             int64_t q_pos0, int64_t chunk_len, float softmax_scale, void* out,
                             const int64_t* os, void* workspace, int64_t workspace_bytes,
                             void* stream) {
    attn::Params p;
    AttnPlan plan;
    bool empty = false;
    int rc = attn_setup(fmt, q, qs, B, Lq, H, D, kc, vc, cs, ks, vs, ss, cache_cap, kv_len, cache_valid,
                        cache_valid_stride, kcur, vcur, curs, cur_len, cur_valid, cur_valid_stride, q_pos0,
                        chunk_len, softmax_scale, out, os, &p, &plan, &empty);
    if (rc != HN_OK || empty) return rc;
    const int64_t need = plan_workspace(plan, B, Lq, H);
    HN_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned(workspace, 16))), HN_E_ARG,
               "hn_attn_fp8kv: workspace smaller than hn_attn_fp8kv_workspace_size() or misaligned");
    return attn_run(p, plan, B, Lq, workspace, (hipStream_t)stream);
}

// ---------------------------------------------------------------------------
// hn_attn_fp8kv_noalloc: hn_attn_fp8kv with the split-key workspace in a
// file-scope device array, for callers that cannot allocate. Each GPU holds
// its own copy of `scratch` until the process ends. Host code never passes the
// array's name (a host-side stand-in) to a kernel: the device address comes
// from hipGetSymbolAddress, looked up once per device with that device current.
// Every call on a device shares its scratch, so calls that overlap on one GPU
// race; the kernels write every partial they read, so nothing needs clearing.
// Size: a split launch keeps at most 2 workgroups per CU in one round, each
// with 128 query rows of (128 + 2) fp32 partials, so a call needs at most
// 2 * CUs * 128 * 130 * 4 bytes: 34.1 MB on MI355X's 256 CUs.
constexpr int64_t NOALLOC_SCRATCH_BYTES = 40ll << 20;
static __device__ __align__(256) uint8_t scratch[NOALLOC_SCRATCH_BYTES];

static std::mutex g_scratch_mu;
static void* g_scratch_ptr[64] = {};

static int scratch_for_current_device(void** out) {
    int dev = -1;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) {
        (void)hipGetLastError();
        return fail(HN_E_DEVICE, "hn_attn_fp8kv_noalloc: no usable current device");
    }
    std::lock_guard<std::mutex> lock(g_scratch_mu);
    if (g_scratch_ptr[dev] == nullptr) {
        void* ptr = nullptr;
        const hipError_t e = hipGetSymbolAddress(&ptr, HIP_SYMBOL(scratch));
        if (e != hipSuccess || ptr == nullptr) {
            (void)hipGetLastError();
            set_error("hn_attn_fp8kv_noalloc: hipGetSymbolAddress of the scratch array failed on device %d: %s",
                      dev, hipGetErrorString(e));
            return HN_E_DEVICE;
        }
        g_scratch_ptr[dev] = ptr;
    }
    *out = g_scratch_ptr[dev];
    return HN_OK;
}

extern "C" int64_t hn_attn_fp8kv_noalloc_scratch_bytes(void) { return NOALLOC_SCRATCH_BYTES; }

extern "C" int hn_attn_fp8kv_noalloc(int fmt, const void* q, const int64_t* qs, int64_t B, int64_t Lq,
                                     int64_t H, int64_t D, const void* kc, const void* vc,
                                     const int64_t* cs, const float* ks, const float* vs,
                                     const int64_t* ss, int64_t cache_cap, int64_t kv_len,
                                     const uint8_t* cache_valid, int64_t cache_valid_stride,
                                     const void* kcur, const void* vcur, const int64_t* curs,
                                     int64_t cur_len, const uint8_t* cur_valid,
                                     int64_t cur_valid_stride, int64_t q_pos0, int64_t chunk_len,
                                     float softmax_scale, void* out, const int64_t* os,
                                     void* stream) {
    attn::Params p;
    AttnPlan plan;
    bool empty = false;
    int rc = attn_setup(fmt, q, qs, B, Lq, H, D, kc, vc, cs, ks, vs, ss, cache_cap, kv_len, cache_valid,
                        cache_valid_stride, kcur, vcur, curs, cur_len, cur_valid, cur_valid_stride, q_pos0,
                        chunk_len, softmax_scale, out, os, &p, &plan, &empty);
    if (rc != HN_OK || empty) return rc;
    const int64_t need = plan_workspace(plan, B, Lq, H);
    if (need > NOALLOC_SCRATCH_BYTES) {
        set_error("hn_attn_fp8kv_noalloc: these sizes need %lld bytes of split-key scratch, more than the "
                  "%lld the library holds per device; call hn_attn_fp8kv with a workspace",
                  (long long)need, (long long)NOALLOC_SCRATCH_BYTES);
        return HN_E_ARG;
    }
    void* ws = nullptr;
    if (need > 0) {
        rc = scratch_for_current_device(&ws);
        if (rc != HN_OK) return rc;
    }
    return attn_run(p, plan, B, Lq, ws, (hipStream_t)stream);
}
