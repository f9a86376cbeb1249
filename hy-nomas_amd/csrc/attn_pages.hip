// Attention over a paged quantized KV cache (gfx950): the queries of every sequence
// against its own tokens, page by page, then the bf16 tail; O = softmax(Q K^T scale) V
// and the rows' log-sum-exp. K, V = bf16(code * scale), as in attn_fp8kv.hip.
#include "attn_pages.h"

namespace hn {
namespace attn {

typedef float f32x4_ __attribute__((ext_vector_type(4)));

// A value that is the same in every lane, as a scalar.
HN_DEVICE int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// A workgroup of NW waves takes 32 NW keys at a time, a unit. Items are dealt out in units
// of four waves.
constexpr int UNIT = 128;

HN_DEVICE int seq_len(const PageParams& p, int b) { return seq_len(p.lens, b, p.width, p.shift); }

// Units of an item: of the cache, of the tail; one at least (a row without keys is written too).
HN_DEVICE int units_of(int keys, int unit) { return (keys + unit - 1) / unit; }
HN_DEVICE int item_units(const PageParams& p, int b, int unit) {
    const int n = units_of(seq_len(p, b), unit) + units_of(p.cur_len, unit);
    return n > 0 ? n : 1;
}

HN_DEVICE uint32_t wave_scan(uint32_t v) {  // inclusive, over the wave
#define HN_SCAN(CTRL, ROWS) \
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false)
    HN_SCAN(0x111, 0xf);  // from 1, 2, 4 and 8 lanes before in the row of 16
    HN_SCAN(0x112, 0xf);
    HN_SCAN(0x114, 0xf);
    HN_SCAN(0x118, 0xf);
    HN_SCAN(0x142, 0xa);  // the row before's last lane
    HN_SCAN(0x143, 0xc);  // the first half's last lane
#undef HN_SCAN
    return v;
}

// Where the items lie on the line of all units: sequence after sequence, in each head
// after head, run after run. Up to 64 sequences are held in a register of the wave, a lane
// each; more are read again where they are needed.
template <int U>
struct Line {
    const PageParams& p;
    uint32_t per, total;
    int mine;        // lane's sequence: units of an item
    uint32_t end;    // and the line's up to its last item
    HN_DEVICE explicit Line(const PageParams& pp) : p(pp), per((uint32_t)(pp.H * pp.runs)), total(0) {
        const int lane = threadIdx.x & 63;
        for (int i0 = 0; i0 < p.B; i0 += 64) {
            mine = i0 + lane < p.B ? item_units(p, i0 + lane, U) : 0;
            end = wave_scan((uint32_t)mine) * per;
            total += (uint32_t)__builtin_amdgcn_readlane((int)end, 63);
        }
    }
    // The sequence of unit u, its first unit on the line, the units of each of its items.
    HN_DEVICE void find(uint32_t u, int& b, uint32_t& start, int& n) const {
        const int lane = threadIdx.x & 63;
        uint32_t before = 0;
        b = 0;
        start = 0;
        n = 1;
        for (int i0 = 0; i0 < p.B; i0 += 64) {
            const int m = p.B <= 64 ? mine : i0 + lane < p.B ? item_units(p, i0 + lane, U) : 0;
            const uint32_t e = p.B <= 64 ? end : wave_scan((uint32_t)m) * per;
            const uint64_t past = __ballot(before + e > u);
            if (past) {
                const int l = __builtin_ctzll(past);
                b = i0 + l;
                n = __builtin_amdgcn_readlane(m, l);
                start = before + (uint32_t)__builtin_amdgcn_readlane((int)e, l) - (uint32_t)n * per;
                return;
            }
            before += (uint32_t)__builtin_amdgcn_readlane((int)e, 63);
        }
    }
    // Of sequence b: its first unit on the line, the units of each of its items.
    HN_DEVICE void place(int b, uint32_t& start, int& n) const {
        if (p.B <= 64) {
            n = __builtin_amdgcn_readlane(mine, b);
            start = (uint32_t)__builtin_amdgcn_readlane((int)end, b) - (uint32_t)n * per;
            return;
        }
        const int lane = threadIdx.x & 63;
        uint32_t before = 0;
        for (int i = lane; i < b; i += 64) before += (uint32_t)item_units(p, i, U);
        start = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(before), 63) * per;
        n = uniform(item_units(p, b, U));
    }
    HN_DEVICE uint32_t share() const { return (total + (uint32_t)p.wgs - 1) / (uint32_t)p.wgs; }
};

HN_DEVICE f32x4_ mfma16_bf16(const bf16x8& a, const bf16x8& b, const f32x4_& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// What a wave's lanes have written to LDS before is there for its other lanes after, and what
// they have read is read. It binds the compiler: the wave's LDS instructions run in their
// order as it is, and the kernels are compiled to the same ones with it.
HN_DEVICE void wave_exchange() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

// How far (log2) a logit may pass the point that a row's probabilities refer to.
constexpr float TOP_HIGH = 8.0f;

// ---------------------------------------------------------------------------
// Few rows against many keys: single tokens, drafted ones, grouped heads. The read of
// the codes is the cost (32 tokens of 8 x 4 heads over up to 16384 keys, 625 MB: 110 us,
// 5.7 TB/s; a kernel that only reads these lines 5.9; 20 rows, 321 MB: 64 to 79 us, the
// dequantization then takes 56 % of the vector unit's cycles). A workgroup holds 16 RB rows
// of one cached head; its four waves take 32-key blocks in turn, each on its own, without
// barriers: S^T = K Q^T and O^T += V^T P^T on 16 x 16 x 32 products whose operands are
// formed in registers. Three waves a SIMD for 16 rows (four spill: 153 us against 125), two
// for 32. With g = lane / 16, r = lane % 16:
//   K operand of keys 16 t + r: the lane has dims 16 g .. + 15 and 64 + 16 g .. + 15 of
//     the key; product s contracts dims 64 (s / 2) + 16 g + 8 (s % 2) + {0..7}, and Q is
//     loaded the same way. The codes pass through the wave's own tile in LDS, so that the
//     loads cover whole lines and pass the caches by.
//   S^T leaves the lane keys 16 t + 4 g + {0..3} of row r: as they stand they are the P
//     operand, slots j < 4 being keys 4 g + j and j >= 4 keys 16 + 4 g + j - 4.
//   V^T operand: for those eight keys the lane loads dims 8 r .. + 7; product db holds dim
//     8 r + db, so that O^T leaves the lane dims 32 g .. + 31 of row r.
// The four waves meet in LDS at the end of an item.
template <int RB>
struct Rows {
    f32x4_ o[RB][8];
    float m[RB], nm[RB], l[RB];
};

// Probabilities are held as the sum of two bf16 (2^-17 relative): V^ is bf16 as it stands,
// where as fp16 it would take one more instruction a value, and the matrix unit has room
// for the second product.
// Loads go through descriptors of a block's rows in its page: a lane has one offset for
// its K rows and one for its V rows, what differs between its loads is a scalar. K is
// asked for again as soon as its operands are formed, V once the product has them, so
// that one set of registers holds a block and its successor is in flight.
struct Probs {
    bf16x8 hi, lo;
};

HN_DEVICE void weigh(const bf16x8& v, const Probs& p, f32x4_& o) {
    o = mfma16_bf16(v, p.hi, o);
    o = mfma16_bf16(v, p.lo, o);
}

struct PageRegs {  // codes of a 32-key block
    uint4 k[4];    // load i: dims 16 (lane % 8) .. of key 8 i + lane / 8
    uint2 v[8];
    float ks[2], vs[8];
};

constexpr int K_TILE = 32 * D;  // bytes of a block's K codes in LDS
constexpr int ONCE = 2;         // loads that pass the caches by (nt): whole lines that nothing reads again

struct Block {
    __amdgpu_buffer_rsrc_t k, v, ks, vs;
    int first, left;  // its first token; keys from there on that the sequence has (<= 0: none)
};

//
// The units of all items are dealt out evenly, whatever the sequences' lengths, and parts of
// an item are joined by a second kernel; or (WHOLE) a workgroup has an item.
template <int FMT, int RB, bool SV, int NW, bool WHOLE>
__global__ __launch_bounds__(64 * NW, NW == 4 && RB == 1 ? 3 : 2) void attn_pages_kernel(PageParams p) {
    constexpr int R = 16 * RB, PITCH = D + 4, UNIT = 32 * NW;
    __shared__ __attribute__((aligned(16))) float so[NW][R][PITCH];
    static_assert(sizeof(so[0]) >= K_TILE, "a wave's K codes fit where its result goes");
    __shared__ float sml[NW][R][2];
    const int id = blockIdx.x;
    const int wg = (id & 7) * p.per_xcd + (id >> 3);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    const int per = p.H * p.runs;

    uint32_t u0, u1, start;   // this workgroup's units; the current sequence's first
    int b, n;
    if constexpr (WHOLE) {
        if (wg >= p.B * per) return;
        b = wg / per;
        n = uniform(item_units(p, b, UNIT));
        start = 0;
        u0 = (uint32_t)(wg - b * per) * (uint32_t)n;
        u1 = u0 + (uint32_t)n;
    } else {
        if (wg >= p.wgs) return;
        const Line<UNIT> line(p);
        const uint32_t share = line.share();
        u0 = (uint32_t)wg * share;
        u1 = u0 + share < line.total ? u0 + share : line.total;
        if (u0 >= u1) return;
        line.find(u0, b, start, n);
    }
    const uint32_t range0 = u0;
    const float c = p.scale_log2;

    while (u0 < u1) {
        if (u0 - start >= (uint32_t)n * (uint32_t)per) {  // the next sequence
            start += (uint32_t)n * (uint32_t)per;
            ++b;
            n = uniform(item_units(p, b, UNIT));
            continue;
        }
        const int item = (int)((u0 - start) / (uint32_t)n);   // h runs + run
        const uint32_t item0 = start + (uint32_t)item * (uint32_t)n;
        const int lo = (int)(u0 - item0), hi = min(n, (int)(u1 - item0));
        const int h = item / p.runs, run = item - h * p.runs;
        const int row0 = run * R, rows = min(R, p.rows - row0);
        const int len = uniform(seq_len(p, b)), nc = units_of(len, UNIT);

        bf16x8 qf[RB][4];
        int lim[RB];           // this lane's rows see cached tokens below
        int lim_all = len;     // all rows do
        const int before = p.causal ? seen_before(p, b, len) : len;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const int r = row0 + min(16 * rb + r16, rows - 1), qi = r / p.G;
            const uint16_t* src = p.q + b * p.qs0 + qi * p.qs1 + (int64_t)(h * p.G + r - qi * p.G) * p.qs2 + 16 * g;
#pragma unroll
            for (int s = 0; s < 4; ++s)
                qf[rb][s] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(src + 64 * (s >> 1) + 8 * (s & 1)));
            lim[rb] = p.causal ? min(before + qi, len) : len;
        }
        if (p.causal) lim_all = min(before + row0 / p.G, len);
        Rows<RB> st;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            st.m[rb] = -INFINITY;
            st.nm[rb] = 0.0f;
            st.l[rb] = 0.0f;
#pragma unroll
            for (int db = 0; db < 8; ++db) st.o[rb][db] = (f32x4_){0.0f, 0.0f, 0.0f, 0.0f};
        }

        // Probabilities of a block's logits s[rb][t] (masked ones -inf), as the P operand.
        auto probs = [&](f32x4_ (&s)[RB][2], Probs (&pf)[RB]) __attribute__((always_inline)) {
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                float mx = -INFINITY;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[rb][t][i]);
                if (__any(mx * c > st.m[rb] + TOP_HIGH)) {
                    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
                    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                    const float mnew = fmaxf(st.m[rb], mx * c);
                    const float a = st.m[rb] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(st.m[rb] - mnew);
                    st.m[rb] = mnew;
                    st.nm[rb] = mnew == -INFINITY ? 0.0f : -mnew;
                    st.l[rb] *= a;
#pragma unroll
                    for (int db = 0; db < 8; ++db) st.o[rb][db] *= a;
                }
                uint32_t x[4], y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rb][e >> 1][2 * (e & 1)], c, st.nm[rb]));
                    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rb][e >> 1][2 * (e & 1) + 1], c, st.nm[rb]));
                    x[e] = pack_bf16(p0, p1);
                    y[e] = pack_bf16(p0 - bf16_lo(x[e]), p1 - bf16_hi(x[e]));
                    st.l[rb] += p0 + p1;
                }
                pf[rb].hi = __builtin_bit_cast(bf16x8, make_uint4(x[0], x[1], x[2], x[3]));
                pf[rb].lo = __builtin_bit_cast(bf16x8, make_uint4(y[0], y[1], y[2], y[3]));
            }
        };

        // ---- cached keys
        const ScalarInts row_table = scalar_ints(p.table + b * p.ts0);
        const int end = NW * min(hi, nc);
        // A block's table entry is a scalar load, asked for a block ahead (a vector load's wait
        // would be for every load before it, the prefetched codes among them).
        auto entry = [&](int blk) __attribute__((always_inline)) {
            return row_table[min((32 * blk) >> p.shift, max(p.width - 1, 0))];
        };
        const int span_c = 31 * (int)p.cs1 + D, span_s = (31 * (int)p.ss1 + 1) * 4, in_page = (1 << p.shift) - 1;
        const uint8_t *kh = p.kc + h * p.cs2, *vh = p.vc + h * p.cs2;
        const float *ksh = p.ks + h * p.ss2, *vsh = p.vs + h * p.ss2;
        auto place = [&](int blk, int e) __attribute__((always_inline)) {
            Block x;
            x.first = blk * 32;
            x.left = blk < end ? len - x.first : 0;
            if ((uint32_t)e >= (uint32_t)p.pages) x.left = 0;  // no such page: no keys
            const int page = x.left > 0 ? e : 0;
            const int64_t slot = x.first & in_page;
            const int64_t ca = page * p.cs0 + slot * p.cs1, sa = page * p.ss0 + slot * p.ss1;
            const int cb = x.left > 0 ? span_c : 0, sb = x.left > 0 ? span_s : 0;
            x.k = tile_rsrc(kh + ca, cb);
            x.v = tile_rsrc(vh + ca, cb);
            x.ks = tile_rsrc(ksh + sa, sb);
            x.vs = tile_rsrc(vsh + sa, sb);
            return x;
        };
        PageRegs x;
        const uint32_t cs1 = (uint32_t)p.cs1, ss1 = 4u * (uint32_t)p.ss1;
        const uint32_t off_k = (lane >> 3) * cs1 + 16 * (lane & 7), off_v = 4 * g * cs1 + 8 * r16, off_ks = r16 * ss1,
                       off_vs = 4 * g * ss1;
        uint8_t* const kt = reinterpret_cast<uint8_t*>(&so[wave][0][0]);  // (this wave's alone until the waves meet)
        uint8_t* const kt_in = kt + (lane >> 3) * D + 16 * ((lane & 7) ^ (lane >> 3));
        auto load_k = [&](const Block& y) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
                x.ks[t] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(y.ks, off_ks, 16 * t * ss1, 0));
#pragma unroll
            for (int i = 0; i < 4; ++i)
                x.k[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(y.k, off_k, 8 * i * cs1, ONCE));
        };
        auto load_v = [&](const Block& y) __attribute__((always_inline)) {
            if constexpr (SV) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const uint4 w = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(y.vs, off_vs, 64 * t, 0));
                    x.vs[4 * t] = __uint_as_float(w.x);
                    x.vs[4 * t + 1] = __uint_as_float(w.y);
                    x.vs[4 * t + 2] = __uint_as_float(w.z);
                    x.vs[4 * t + 3] = __uint_as_float(w.w);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t key = 16 * (j >> 2) + (j & 3);  // + 4 g
                x.v[j] = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(y.v, off_v, key * cs1, ONCE));
                if constexpr (!SV)
                    x.vs[j] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(y.vs, off_vs, key * ss1, 0));
            }
        };
        int blk = NW * lo + wave;
        int e = blk < end ? entry(blk) : 0, e1 = blk + NW < end ? entry(blk + NW) : 0;
        Block now = place(blk, e);
        // (in the loop's order, by which each wait knows its loads)
        load_k(now);
        __builtin_amdgcn_sched_barrier(0);
        load_v(now);
        __builtin_amdgcn_sched_barrier(0);
        for (; blk < end; blk += NW) {
            const Block next = place(blk + NW, e1);
            e1 = blk + 2 * NW < end ? entry(blk + 2 * NW) : 0;
            // K codes through the wave's own LDS tile (chunk c of row r at c ^ r % 8)
            uint4 kx[2][2];
            const float ks[2] = {x.ks[0], x.ks[1]};
#pragma unroll
            for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(kt_in + 8 * i * D) = x.k[i];
            wave_exchange();
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    kx[t][e] = *reinterpret_cast<const uint4*>(kt + (16 * t + r16) * D + 16 * ((g + 4 * e) ^ (r16 & 7)));
            wave_exchange();  // (the next block's codes, or the item's result, go there)
            __builtin_amdgcn_sched_barrier(0);
            load_k(next);
            __builtin_amdgcn_sched_barrier(0);
            f32x4_ s[RB][2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) s[rb][t] = (f32x4_){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int sl = 0; sl < 4; ++sl) {
                    uint32_t d[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const f32x2 f = codes2_f32<FMT>(word(kx[t][sl >> 1], 2 * (sl & 1) + (e >> 1)), e & 1);
                        d[e] = pack_bf16(f[0] * ks[t], f[1] * ks[t]);
                    }
                    const bf16x8 kf = __builtin_bit_cast(bf16x8, make_uint4(d[0], d[1], d[2], d[3]));
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) s[rb][t] = mfma16_bf16(kf, qf[rb][sl], s[rb][t]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (now.left > 0) {
                if (now.first + 32 > lim_all) {
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                        for (int t = 0; t < 2; ++t)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (now.first + 16 * t + 4 * g + i >= lim[rb]) s[rb][t][i] = -INFINITY;
                }
                if (now.left < 32) {  // what lies behind the sequence's end meets no product
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (16 * (j >> 2) + 4 * g + (j & 3) >= now.left) {
                            x.v[j] = make_uint2(0u, 0u);
                            x.vs[j] = 0.0f;
                        }
                }
                Probs pf[RB];
                probs(s, pf);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    f32x2 f[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        f[j] = codes2_f32<FMT>(e & 2 ? x.v[j].y : x.v[j].x, e & 1);
                        f[j][0] *= x.vs[j];
                        f[j][1] *= x.vs[j];
                    }
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const bf16x8 vf = __builtin_bit_cast(
                            bf16x8, make_uint4(pack_bf16(f[0][w], f[1][w]), pack_bf16(f[2][w], f[3][w]),
                                               pack_bf16(f[4][w], f[5][w]), pack_bf16(f[6][w], f[7][w])));
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb) weigh(vf, pf[rb], st.o[rb][2 * e + w]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            load_v(next);
            __builtin_amdgcn_sched_barrier(0);
            now = next;
        }
        // ---- the tail
        for (int u = max(lo, nc); u < hi; ++u) {
            const int first = (u - nc) * UNIT + 32 * wave, left = p.cur_len - first;
            if (left <= 0) break;
            const int64_t at = b * p.us0 + h * p.us2;
            bool ok = (lane & 31) < left;
            if (p.uvalid && ok) ok = p.uvalid[b * p.uvs + first + (lane & 31)] != 0;
            const uint32_t live = (uint32_t)__ballot(ok);
            if (live == 0) continue;
            f32x4_ s[RB][2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const uint16_t* kp = p.kcur + at + (int64_t)(first + min(16 * t + r16, left - 1)) * p.us1 + 16 * g;
                uint4 kx[4];
#pragma unroll
                for (int sl = 0; sl < 4; ++sl) kx[sl] = *reinterpret_cast<const uint4*>(kp + 64 * (sl >> 1) + 8 * (sl & 1));
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    s[rb][t] = (f32x4_){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int sl = 0; sl < 4; ++sl)
                        s[rb][t] = mfma16_bf16(__builtin_bit_cast(bf16x8, kx[sl]), qf[rb][sl], s[rb][t]);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (!((live >> (16 * t + 4 * g + i)) & 1u)) s[rb][t][i] = -INFINITY;
                }
            }
            uint4 vx[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int key = 16 * (j >> 2) + 4 * g + (j & 3);
                vx[j] = make_uint4(0u, 0u, 0u, 0u);
                if ((live >> key) & 1u)
                    vx[j] = *reinterpret_cast<const uint4*>(p.vcur + at + (int64_t)(first + key) * p.us1 + 8 * r16);
            }
            Probs pf[RB];
            probs(s, pf);
#pragma unroll
            for (int db = 0; db < 8; ++db) {
                uint32_t y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t a = word(vx[2 * e], db >> 1), z = word(vx[2 * e + 1], db >> 1);
                    y[e] = __builtin_amdgcn_perm(z, a, db & 1 ? 0x07060302u : 0x05040100u);  // high or low halves
                }
                const bf16x8 vf = __builtin_bit_cast(bf16x8, make_uint4(y[0], y[1], y[2], y[3]));
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) weigh(vf, pf[rb], st.o[rb][db]);
            }
        }
        // ---- the waves meet
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            float l = st.l[rb];
            l += __shfl_xor(l, 16, 64);
            l += __shfl_xor(l, 32, 64);
            const int r = 16 * rb + r16;
            if (r < rows) {
                float* dst = &so[wave][r][32 * g];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        *reinterpret_cast<float4*>(dst + 8 * i + 4 * e) =
                            make_float4(st.o[rb][4 * e][i], st.o[rb][4 * e + 1][i], st.o[rb][4 * e + 2][i], st.o[rb][4 * e + 3][i]);
                if (g == 0) {
                    sml[wave][r][0] = st.m[rb];
                    sml[wave][r][1] = l;
                }
            }
        }
        __syncthreads();
        const bool done = lo == 0 && hi == n;
        const int64_t part = (int64_t)wg * 2 + (item0 < range0 ? 0 : 1);
        for (int at = threadIdx.x; at < rows * (D / 4); at += 64 * NW) {
            const int r = at / (D / 4), d = (at % (D / 4)) * 4;
            float m = sml[0][r][0];
#pragma unroll
            for (int w = 1; w < NW; ++w) m = fmaxf(m, sml[w][r][0]);
            const float base = m == -INFINITY ? 0.0f : m;
            float den = 0.0f;
            float4 num = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float a = __builtin_amdgcn_exp2f(sml[w][r][0] - base);
                const float4 y = *reinterpret_cast<const float4*>(&so[w][r][d]);
                den = __builtin_fmaf(sml[w][r][1], a, den);
                num.x = __builtin_fmaf(y.x, a, num.x);
                num.y = __builtin_fmaf(y.y, a, num.y);
                num.z = __builtin_fmaf(y.z, a, num.z);
                num.w = __builtin_fmaf(y.w, a, num.w);
            }
            if (done) {
                const int rr = row0 + r, qi = rr / p.G, hq = h * p.G + rr - qi * p.G;
                const float inv = den != 0.0f ? 1.0f / den : 0.0f;
                *reinterpret_cast<uint2*>(p.out + b * p.os0 + qi * p.os1 + hq * p.os2 + d) =
                    make_uint2(pack_bf16(num.x * inv, num.y * inv), pack_bf16(num.z * inv, num.w * inv));
                if (d == 0)
                    p.lse[((int64_t)b * p.H * p.G + hq) * p.Lq + qi] =
                        den != 0.0f ? (m + __builtin_amdgcn_logf(den)) * 0.6931471805599453f : -INFINITY;
            } else {
                *reinterpret_cast<float4*>(p.ws_o + (part * p.pitch + r) * D + d) = num;
                if (d == 0) *reinterpret_cast<float2*>(p.ws_ml + (part * p.pitch + r) * 2) = make_float2(m, den);
            }
        }
        __syncthreads();
        u0 = item0 + (uint32_t)hi;
    }
}

// ---------------------------------------------------------------------------
// Many rows: the 8-wave, three-stage half-tile loop of attn_fp8kv.hip (256 rows a
// workgroup, one barrier a tile), its cache tiles from the pages through descriptors of
// their own rows, its denominator from the fp32 probabilities. The tiles of all items are
// dealt out evenly to as many workgroups as there are CUs, so that neither the sequences'
// lengths nor a last round of workgroups leaves any idle (two sequences' 3600 queries x 24
// heads over 21600 keys and the tail: 2.40 ms, 0.93 PFLOP/s; by runs of 128 rows on 4
// waves 2.83); parts meet in pages_join_kernel. An item costs 11 us beside its tiles (2.4 us
// each), whose products are those of 256 rows however many are valid. Causal items count
// every key, though their first rows see few: the largest share of computed tiles is 1.2 to
// 1.95 times the mean (24 heads, 16384 tokens: 2.96 ms where the products take 1.29). The
// part of a tile past a length or a tail, and a page that is none, read as zeros and are
// masked by the tile's 64-bit word.
constexpr int TILE_WAVES = 8;
constexpr int TILE_ROWS = Shape<TILE_WAVES>::BQ;

template <int FMT, bool MASK, bool CAUSAL>
__global__ __launch_bounds__(64 * TILE_WAVES, 1) void attn_page_tiles_kernel(PageParams p, Params t_) {
    constexpr int NW = TILE_WAVES, NS = 3;
    __shared__ __attribute__((aligned(16))) uint8_t smem[NS * STAGE + 2 * SB_FLOATS * 4];
    float* const sbuf = reinterpret_cast<float*>(smem + NS * STAGE);  // [2][128]
    const int id = blockIdx.x;
    const int wg = (id & 7) * p.per_xcd + (id >> 3);
    if (wg >= p.wgs) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5, qd = threadIdx.x & 15;
    const int per = p.H * p.runs;
    uint32_t u0, u1, start;
    int b, n;
    {
        const Line<BKV> line(p);
        const uint32_t share = line.share();
        u0 = (uint32_t)wg * share;
        u1 = u0 + share < line.total ? u0 + share : line.total;
        if (u0 >= u1) return;
        line.find(u0, b, start, n);
    }
    const uint32_t range0 = u0;
    const float c = p.scale_log2;
    const int cur_len = p.cur_len;
    const LaneOffs<NW> lo = lane_offsets<NW>(t_);
    const TailOffs<NW> to = tail_offsets<NW>(t_);
    const bool tail_ok = ((int64_t)cur_len * p.us1 + D) * 2 < ((int64_t)1 << 31);
    const uint32_t ka_off = col * KROW + 16 * half, va_off = K_BYTES + col * VTROW + 16 * half;

    while (u0 < u1) {
        if (u0 - start >= (uint32_t)n * (uint32_t)per) {  // the next sequence
            start += (uint32_t)n * (uint32_t)per;
            ++b;
            n = uniform(item_units(p, b, BKV));
            continue;
        }
        const int item = (int)((u0 - start) / (uint32_t)n);  // h runs + run
        const uint32_t item0 = start + (uint32_t)item * (uint32_t)n;
        const int h = item / p.runs, run = item - h * p.runs;
        const int t_begin = (int)(u0 - item0), hi = min(n, (int)(u1 - item0));
        const int len = uniform(seq_len(p, b)), nc = units_of(len, BKV), n_all = nc + units_of(cur_len, BKV);
        const int row = run * TILE_ROWS + wave * QW + col;
        const bool qvalid = row < p.rows;
        const int rr = qvalid ? row : p.rows - 1, qi = rr / p.G, hq = h * p.G + rr - qi * p.G;
        // CAUSAL: this lane's row sees tokens below lim, every row those below lim_all, and
        // none those from lim_end on.
        int lim = 0, lim_all = 0, t_end = min(hi, n_all);  // (an item without a key has a unit, but no tile)
        if constexpr (CAUSAL) {
            const int before = seen_before(p, b, len);
            lim = min(before + qi, len);
            lim_all = min(before + run * TILE_ROWS / p.G, len);
            const int lim_end = before + min(run * TILE_ROWS + TILE_ROWS - 1, p.rows - 1) / p.G;
            t_end = min(t_end, units_of(max(lim_end, 0), BKV));
        }
        bf16x8 qf[8];
        {
            const uint16_t* src = p.q + b * p.qs0 + qi * p.qs1 + hq * p.qs2 + half * 8;
#pragma unroll
            for (int sl = 0; sl < 8; ++sl)
                qf[sl] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(src + 16 * sl));
        }
        f32x16 o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int v = 0; v < 16; ++v) o[i][v] = 0.0f;
        Run run_{-INFINITY, 0.0f, 0.0f};

        // Keys of tile t, and where its loads start.
        struct Place {
            TileBase src;
            int count;
        };
        const ScalarInts row_table = scalar_ints(p.table + b * p.ts0);
        const int in_page = (1 << p.shift) - 1;
        auto cache_tile = [&](int t) __attribute__((always_inline)) {
            Place g;
            const int first = t * BKV;
            int page = -1;
            if (t < nc && t < t_end) page = row_table[first >> p.shift];
            const bool there = (uint32_t)page < (uint32_t)p.pages;
            g.count = there ? min(BKV, len - first) : 0;
            g.src = tile_base(t_, there ? page : 0, h, first & in_page, g.count);
            return g;
        };
        auto tail_keys = [&](int t) __attribute__((always_inline)) {
            const int left = t < t_end ? cur_len - (t - nc) * BKV : 0;
            return left >= BKV ? BKV : left > 0 ? left : 0;
        };
        auto tail_rsrc = [&](const uint16_t* base, int64_t first, int64_t rows) __attribute__((always_inline)) {
            return tile_rsrc(base + b * p.us0 + h * p.us2 + first * p.us1, rows > 0 ? ((rows - 1) * p.us1 + D) * 2 : 0);
        };
        __amdgpu_buffer_rsrc_t tk = tail_rsrc(p.kcur, 0, tail_ok ? cur_len : 0),
                               tv = tail_rsrc(p.vcur, 0, tail_ok ? cur_len : 0);
        CacheRegs<NW> regs;
        regs.s = 0.0f;
        TailRegs<NW> tr;
        uint32_t vbits = 0xffffffffu;  // MASK: validity bytes of this thread's four V keys
        auto fetch_cache_k = [&](const Place& g) __attribute__((always_inline)) { load_k<NW, false>(lo, regs, g.src, g.count); };
        auto fetch_tail = [&](int t) __attribute__((always_inline)) {
            const int count = tail_keys(t);
            const int64_t first = (int64_t)(t - nc) * BKV;
            uint32_t co = count > 0 ? (uint32_t)(first * p.us1 * 2) : 0x80000000u;
            if (!tail_ok && count > 0) {
                tk = tail_rsrc(p.kcur, first, count);
                tv = tail_rsrc(p.vcur, first, count);
                co = 0;
            }
            load_tail_span_k<NW, MASK>(t_, b, to, tk, co, first, first + count, tr);
            load_tail_span_v<NW>(to, tv, co, tr);
            if constexpr (MASK) {
                vbits = 0u;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int key = quad_key(qd, j);
                    if (key < count && (!p.uvalid || p.uvalid[b * p.uvs + first + key] != 0)) vbits |= 0xffu << (8 * j);
                }
            }
        };
        // What a masked key's V holds meets no product.
        auto clear_tail_v = [&]() __attribute__((always_inline)) {
            if constexpr (MASK)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (!((vbits >> (8 * j)) & 1u)) tr.v[j][0] = tr.v[j][1] = 0u;
        };
        // The keys of tile t that take part, in the stage that holds it.
        auto word_of = [&](int t, int count, const uint8_t* st) __attribute__((always_inline)) {
            const uint64_t all = count >= BKV ? ALL_KEYS : (1ull << count) - 1;
            if constexpr (MASK)
                if (t >= nc) return tile_mask<true>(st) & all;
            return all;
        };

        if (t_end > t_begin) {
            // ---- prologue: tiles t_begin, + 1 in stages 0, 1, the next one's codes in registers
            int c0 = 0, c1 = 0, c2 = 0;  // keys of tiles t, t + 1, t + 2
            const bool cached = t_begin + 2 < nc;
            if (cached) {  // the three tiles' loads in flight together
                const Place g0 = cache_tile(t_begin), g1 = cache_tile(t_begin + 1), g2 = cache_tile(t_begin + 2);
                CacheRegs<NW> r0, r1;
                r0.s = r1.s = 0.0f;
                load_k<NW, false>(lo, r0, g0.src, g0.count);
                load_v<NW>(lo, r0, g0.src);
                load_k<NW, false>(lo, r1, g1.src, g1.count);
                load_v<NW>(lo, r1, g1.src);
                fetch_cache_k(g2);
                load_v<NW>(lo, regs, g2.src);
                c0 = g0.count;
                c1 = g1.count;
                c2 = g2.count;
                __builtin_amdgcn_s_waitcnt(0);
                if (threadIdx.x < 2 * BKV) {
                    sbuf[threadIdx.x] = r0.s;
                    sbuf[SB_FLOATS + threadIdx.x] = r1.s;
                }
                __syncthreads();
                store_tile<FMT, NW, false>(r0, smem, sbuf);
                store_tile<FMT, NW, false>(r1, smem + STAGE, sbuf + SB_FLOATS);
                __syncthreads();
                if (threadIdx.x < 2 * BKV) sbuf[threadIdx.x] = regs.s;
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if (cached) break;
                const int t = t_begin + k;
                int count = 0;
                if (t < nc) {
                    const Place g = cache_tile(t);
                    count = g.count;
                    fetch_cache_k(g);
                    load_v<NW>(lo, regs, g.src);
                    __builtin_amdgcn_s_waitcnt(0);
                    if (threadIdx.x < 2 * BKV) sbuf[(k & 1) * SB_FLOATS + threadIdx.x] = regs.s;
                    __syncthreads();
                    store_tile<FMT, NW, false>(regs, smem + k * STAGE, sbuf + (k & 1) * SB_FLOATS);
                } else {
                    count = tail_keys(t);
                    fetch_tail(t);
                    store_tail_k<NW, MASK>(tr, smem + k * STAGE);
                    clear_tail_v();
                    store_tail_v<NW>(tr, smem + k * STAGE);
                }
                if (k == 0) c0 = count;
                else c1 = count;
            }
            if (!cached) {
                c2 = tail_keys(t_begin + 2);
                fetch_tail(t_begin + 2);
                __builtin_amdgcn_s_waitcnt(0);
            }
            __syncthreads();
            uint64_t mw = word_of(t_begin, c0, smem);
            f32x16 sa = s_block(smem + ka_off, qf), sb;
            float mxa = raw_max(sa), mxb;
            // Masks half kb of tile t, whose largest logit was mx.
            auto masked = [&](f32x16& x, int t, int kb, uint64_t word, float mx) __attribute__((always_inline)) {
                if constexpr (CAUSAL)
                    if ((t + 1) * BKV > lim_all) return mask_raw(x, kb, half, lim - t * BKV, word);
                const uint32_t w = (uint32_t)(word >> (32 * kb));
                return w == ~0u ? mx : mask_word(x, w);
            };
            mxa = masked(sa, t_begin, 0, mw, mxa);
            int t = t_begin, s0 = 0;  // s0: stage of tile t

            // Tile t: S of t + 1 and the write of t + 2 beside its products; KC, FC: tile t + 2
            // (written), t + 3 (asked for) are the cache's.
            auto tile = [&](auto kc, auto fc) __attribute__((always_inline)) {
                constexpr bool KC = decltype(kc)::value, FC = decltype(fc)::value;
                const int u = t - t_begin;
                const int s1 = s0 == NS - 1 ? 0 : s0 + 1, sw = s0 == 0 ? NS - 1 : s0 - 1;
                const uint8_t* st = smem + s0 * STAGE;
                const uint8_t* st1 = smem + s1 * STAGE;
                uint8_t* wst = smem + sw * STAGE;
                const float* wsb = sbuf + (u & 1) * SB_FLOATS;
                Place g3;
                if constexpr (FC) g3 = cache_tile(t + 3);
                const int c3 = FC ? g3.count : tail_keys(t + 3);
                f16x8 pf[2];
                const uint64_t mwn = word_of(t + 1, c1, st1);
                // half 0
                rebase_high(mxa, c, run_, o);
                sb = step_a_lse(sa, c, run_.nm, run_.l, pf, st + ka_off + 32 * KROW, qf);
                if constexpr (KC) {
                    mxb = step_b<FMT, NW, 1>(pf, st + va_off, 0, o, sb, regs, wst, wsb);
                } else {
                    mxb = step_b_with(pf, st + va_off, 0, o, sb, [&](int i) __attribute__((always_inline)) {
                        if (i == 3 || i == 6) store_tail_k_part<NW>(tr, wst, 0, i == 6);
                    });
                    store_tail_mask<NW, MASK>(tr, wst);
                }
                mxb = masked(sb, t, 1, mw, mxb);
                if constexpr (FC) fetch_cache_k(g3);
                // half 1 (on the last tile the S block of "tile t + 1" reads stale LDS; its
                // result is never used)
                rebase_high(mxb, c, run_, o);
                sa = step_a_lse(sb, c, run_.nm, run_.l, pf, st1 + ka_off, qf);
                if constexpr (KC) {
                    mxa = step_b<FMT, NW, 2>(pf, st + va_off, 1, o, sa, regs, wst, wsb);
                } else {
                    clear_tail_v();
                    mxa = step_b_with(pf, st + va_off, 1, o, sa, [&](int i) __attribute__((always_inline)) {
                        if (i & 1) store_tail_v_part<NW>(tr, wst, i >> 1);
                    });
                }
                mxa = masked(sa, t + 1, 0, mwn, mxa);
                if constexpr (FC) {
                    if (threadIdx.x < 2 * BKV) sbuf[((u + 1) & 1) * SB_FLOATS + threadIdx.x] = regs.s;
                    load_v<NW>(lo, regs, g3.src);
                } else {
                    fetch_tail(t + 3);
                }
                __syncthreads();
                s0 = s1;
                mw = mwn;
                c0 = c1;
                c1 = c2;
                c2 = c3;
            };
            const auto yes = std::integral_constant<bool, true>{};
            const auto no = std::integral_constant<bool, false>{};
            // (past the end of the range both kinds are empty: cache_tile and tail_keys say so)
            for (; t < t_end && t + 3 < nc; ++t) tile(yes, yes);
            for (; t < t_end && t + 2 < nc; ++t) tile(yes, no);
            for (; t < t_end; ++t) tile(no, no);
        }
        const float l = run_.l + __shfl_xor(run_.l, 32, 64), m = run_.m;
        if (qvalid) {
            if (t_begin == 0 && hi == n) {
                const float inv = l != 0.0f ? 1.0f / l : 0.0f;
                uint16_t* dst = p.out + b * p.os0 + qi * p.os1 + hq * p.os2;
#pragma unroll
                for (int db = 0; db < 4; ++db)
#pragma unroll
                    for (int vq = 0; vq < 4; ++vq)
                        *reinterpret_cast<uint2*>(dst + db * 32 + vq * 8 + half * 4) =
                            make_uint2(pack_bf16(o[db][vq * 4] * inv, o[db][vq * 4 + 1] * inv),
                                       pack_bf16(o[db][vq * 4 + 2] * inv, o[db][vq * 4 + 3] * inv));
                if (half == 0)
                    p.lse[((int64_t)b * p.H * p.G + hq) * p.Lq + qi] =
                        l != 0.0f ? (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f : -INFINITY;
            } else {
                const int64_t at = ((int64_t)wg * 2 + (item0 < range0 ? 0 : 1)) * p.pitch + wave * QW + col;
                float* dst = p.ws_o + at * D;
#pragma unroll
                for (int db = 0; db < 4; ++db)
#pragma unroll
                    for (int vq = 0; vq < 4; ++vq)
                        *reinterpret_cast<float4*>(dst + db * 32 + vq * 8 + half * 4) =
                            make_float4(o[db][vq * 4], o[db][vq * 4 + 1], o[db][vq * 4 + 2], o[db][vq * 4 + 3]);
                if (half == 0) *reinterpret_cast<float2*>(p.ws_ml + at * 2) = make_float2(m, l);
            }
        }
        __syncthreads();  // (the stages are the next item's)
        u0 = item0 + (uint32_t)hi;
    }
}

// The parts of items that several workgroups computed, joined in their order: with M =
// max m, O = sum 2^(m - M) O / sum 2^(m - M) l. 32 threads a row, 4 dims each, eight parts
// in flight, eight rows of an item a workgroup. Workgroups stand for the items, or (SEAMS)
// for the borders between two workgroups' shares, whichever are fewer: an item is its first
// border's (two branches' frames, 720 items of 256 rows: 40 us by items, 27 by borders). Where
// an item has many parts (ROWS) a workgroup has one row, whose parts its eight groups of
// threads take in turn (one sequence of 100000 keys, 96 parts: 4.4 us, by eight rows 10.2;
// four parts of twenty rows 8.0, by eight rows 4.7).
enum Join { ITEMS, SEAMS, ROWS };
constexpr int MANY_PARTS = 16;

template <int U, Join JOIN>
__global__ __launch_bounds__(256) void pages_join_kernel(PageParams p, int R) {
    const Line<U> line(p);
    const int per = p.H * p.runs, groups = JOIN == ROWS ? p.pitch : (p.pitch + 7) / 8;
    int x = blockIdx.x;
    const int grp = x % groups;
    x /= groups;
    const uint32_t share = line.share();
    uint32_t start;
    int n, b, item;
    if constexpr (JOIN == SEAMS) {
        const uint32_t seam = (uint32_t)(x + 1) * share;
        if (seam >= line.total) return;
        line.find(seam, b, start, n);
        item = (int)((seam - start) / (uint32_t)n);
    } else {
        item = x % per;
        b = x / per;
        line.place(b, start, n);
    }
    const uint32_t i0 = start + (uint32_t)item * (uint32_t)n;
    const uint32_t w0 = i0 / share, w1 = (i0 + (uint32_t)n - 1) / share;
    if (w0 == w1 || (JOIN == SEAMS && (uint32_t)x != w0)) return;  // whole (written already), or another border's
    const int h = item / p.runs, run = item - h * p.runs;
    constexpr uint32_t STEP = JOIN == ROWS ? 8 : 1;
    const int tg = threadIdx.x >> 5, r = JOIN == ROWS ? grp : grp * 8 + tg, row = run * R + r, d = (threadIdx.x & 31) * 4;
    if (r >= p.pitch || row >= p.rows) return;
    float M = -INFINITY, den = 0.0f;
    float4 num = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (uint32_t a0 = w0 + (JOIN == ROWS ? tg : 0); a0 <= w1; a0 += 8 * STEP) {
        float2 ml[8];
        float4 ov[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t w = min(a0 + e * STEP, w1);
            const int64_t part = ((int64_t)w * 2 + (i0 < w * share ? 0 : 1)) * p.pitch + r;
            ml[e] = *reinterpret_cast<const float2*>(p.ws_ml + part * 2);
            ov[e] = *reinterpret_cast<const float4*>(p.ws_o + part * D + d);
            if (a0 + e * STEP > w1) ml[e] = make_float2(-INFINITY, 0.0f);
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
    if constexpr (JOIN == ROWS) {
        __shared__ __attribute__((aligned(16))) float4 so[8][D / 4];
        __shared__ float2 sml[8];
        so[tg][d / 4] = num;
        if (d == 0) sml[tg] = make_float2(M, den);
        __syncthreads();
        if (tg > 0) return;
#pragma unroll
        for (int e = 0; e < 8; ++e) M = fmaxf(M, sml[e].x);
        const float base = M == -INFINITY ? 0.0f : M;
        den = 0.0f;
        num = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float wgt = __builtin_amdgcn_exp2f(sml[e].x - base);
            const float4 y = so[e][d / 4];
            den = fmaf(wgt, sml[e].y, den);
            num.x = fmaf(wgt, y.x, num.x);
            num.y = fmaf(wgt, y.y, num.y);
            num.z = fmaf(wgt, y.z, num.z);
            num.w = fmaf(wgt, y.w, num.w);
        }
    }
    const int qi = row / p.G, hq = h * p.G + row - qi * p.G;
    const float inv = den != 0.0f ? 1.0f / den : 0.0f;
    *reinterpret_cast<uint2*>(p.out + b * p.os0 + qi * p.os1 + hq * p.os2 + d) =
        make_uint2(pack_bf16(num.x * inv, num.y * inv), pack_bf16(num.z * inv, num.w * inv));
    if (d == 0)
        p.lse[((int64_t)b * p.H * p.G + hq) * p.Lq + qi] =
            den != 0.0f ? (M + __builtin_amdgcn_logf(den)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace attn
}  // namespace hn

using namespace hn;

struct PagesPlan {
    int tiles;   // 0: attn_pages_kernel; 4, 8: the tile kernel of as many waves
    int whole;   // of attn_pages_kernel: waves of a workgroup an item; 0: units dealt out
    int rb, runs, wgs, pitch;
    int64_t items;
};

static PagesPlan pages_plan(int64_t B, int64_t Lq, int64_t G, int64_t H, int64_t max_len, int64_t cur_len) {
    PagesPlan pl;
    const int64_t rows = Lq * G;
    // attn_pages_kernel (0), the 4-wave tiles or the 8-wave ones, calls in us. 33 to 64 rows, 0
    // against 4: 64 sequences x 8 heads, 300 keys 44 and 23, 1000 keys 82 to 91 and 47, 4000 155 to
    // 161 and 153; 20000 keys of eight 80 and 100, of two x 24 heads 73 to 78 and 95. 32 rows: 20000
    // keys 50 and 82 to 92. 128 rows, 20000 keys x 2 x 24 heads: 182 and 107, 8-wave 147. More
    // rows, 4 against 8, up to 1000 and 4000 keys: 32 sequences x 8 heads, 300 rows 75 and 108, 209
    // and 229, 1000 rows 187 and 188, 444 and 387; 8 x 8, 600 rows 47 and 67, 117 and 97; up to
    // 2000 keys 39 and 50 (2 x 24, 300 rows), 121 and 119 (8 x 8, 1200), 272 and 247 (4000). The
    // same borders for causal rows.
    const int64_t keys = max_len + cur_len;
    pl.tiles = rows <= 32 || (rows <= 64 && keys > 4096) ? 0 : rows <= 128 || keys <= 2048 ? 4 : attn::TILE_WAVES;
    if (pl.tiles == attn::TILE_WAVES) {
        pl.runs = (int)((rows + attn::TILE_ROWS - 1) / attn::TILE_ROWS);
        pl.items = B * H * pl.runs;
        pl.pitch = (int)(rows < attn::TILE_ROWS ? rows : attn::TILE_ROWS);
        pl.wgs = device_cus();
        pl.whole = 0;
        return pl;
    }
    pl.rb = rows <= 16 ? 1 : 2;
    const int64_t R = 16 * pl.rb;
    pl.runs = (int)((rows + R - 1) / R);
    pl.items = B * H * pl.runs;
    pl.pitch = (int)(rows < R ? rows : R);
    // A workgroup an item: of eight waves where each has few keys and all are resident at once
    // (calls of 8 to 256 items of one to four rows, kernels in us: up to 100 keys 6 against 8.4
    // to 12.4 dealt out and joined, 500 8.2 to 10.6 against 9.1 to 17.1, 1024 11.1 to 16.4 against
    // 11.3 to 24.2, 2048 (eight items) 17.5 against 13.3; twenty rows 500 11.2 against 14.2, 1024
    // 15.3 against 14.6), of four where many items come and go (calls, sequences of n / 8 to n keys
    // and of n, against dealt out: 2048 items of four rows, n 500 37 and 51 against 63 and 67, 2000
    // 112 and 178 against 120 and 192, 4000 224 and 333 against 223 and 353; 512 items 1000 21 and 30
    // against 28 and 35, with eight waves 25; 4000 66 and 88 against 66 and 98, 6000 88 and 128 against
    // 87 and 141; 256 items 2000 23 and 26 against 26 and 34, 4000 39 and 45 against 38 and 55, twenty
    // rows there 50 and 59 against 47 and 55).
    const int64_t units = (max_len + 255) / 256 + (cur_len + 255) / 256, cus = device_cus();
    pl.wgs = (int)((pl.rb == 1 ? 3 : 2) * cus);
    if (pl.items < cus) pl.whole = units * pl.rb <= 4 ? 8 : 0;
    else pl.whole = keys <= (pl.items < 2 * cus ? 2048 : 4096) && pl.items <= 1 << 22 ? 4 : 0;  // (a grid has fewer than 2^32 threads)
    return pl;
}

// SV: the scales of consecutive tokens are consecutive, four to a load.
template <int FMT, int NW, bool WHOLE>
static void launch_pages(int rb, bool sv, const attn::PageParams& p, unsigned blocks, hipStream_t st) {
    if (rb == 1 && sv) attn::attn_pages_kernel<FMT, 1, true, NW, WHOLE><<<blocks, 64 * NW, 0, st>>>(p);
    else if (rb == 1) attn::attn_pages_kernel<FMT, 1, false, NW, WHOLE><<<blocks, 64 * NW, 0, st>>>(p);
    else if (sv) attn::attn_pages_kernel<FMT, 2, true, NW, WHOLE><<<blocks, 64 * NW, 0, st>>>(p);
    else attn::attn_pages_kernel<FMT, 2, false, NW, WHOLE><<<blocks, 64 * NW, 0, st>>>(p);
}

template <int FMT>
static void launch_few(const PagesPlan& pl, bool sv, const attn::PageParams& p, unsigned blocks, hipStream_t st) {
    if (pl.whole == 8) launch_pages<FMT, 8, true>(pl.rb, sv, p, blocks, st);
    else if (pl.whole) launch_pages<FMT, 4, true>(pl.rb, sv, p, blocks, st);
    else launch_pages<FMT, 4, false>(pl.rb, sv, p, blocks, st);
}

template <int FMT>
static void launch_tiles(const attn::PageParams& p, const attn::Params& t, unsigned blocks, hipStream_t st) {
    constexpr int threads = 64 * attn::TILE_WAVES;
    if (p.causal) attn::attn_page_tiles_kernel<FMT, false, true><<<blocks, threads, 0, st>>>(p, t);
    else if (p.uvalid) attn::attn_page_tiles_kernel<FMT, true, false><<<blocks, threads, 0, st>>>(p, t);
    else attn::attn_page_tiles_kernel<FMT, false, false><<<blocks, threads, 0, st>>>(p, t);
}

static bool pages_shape_ok(int64_t B, int64_t Lq, int64_t Hq, int64_t H, int64_t max_len, int64_t cur_len) {
    return B > 0 && Lq > 0 && H > 0 && Hq > 0 && Hq % H == 0 && max_len >= 0 && cur_len >= 0 && B <= 0x7fffffffLL &&
           Lq <= 0x7fffffffLL && Hq <= 0x7fffffffLL && max_len <= 0x3fffffffLL && cur_len <= 0x3fffffffLL &&
           Lq * (Hq / H) <= 0x3fffffffLL;
}

template <int U>
static int join_pages(const PagesPlan& pl, const attn::PageParams& p, int R, hipStream_t st) {
    const int64_t groups = (pl.pitch + 7) / 8;
    if (pl.items * attn::MANY_PARTS <= pl.wgs)
        attn::pages_join_kernel<U, attn::ROWS><<<(unsigned)(pl.items * pl.pitch), 256, 0, st>>>(p, R);
    else if (pl.items < pl.wgs)
        attn::pages_join_kernel<U, attn::ITEMS><<<(unsigned)(pl.items * groups), 256, 0, st>>>(p, R);
    else attn::pages_join_kernel<U, attn::SEAMS><<<(unsigned)((pl.wgs - 1) * groups), 256, 0, st>>>(p, R);
    return check_launch("hn_attn_kv_pages (join)");
}

static int64_t plan_bytes(const PagesPlan& pl, int64_t B, int64_t Lq, int64_t Hq, int64_t H, int64_t max_len,
                          int64_t cur_len) {
    if (pl.tiles == 4) return page_tiles_workspace(B, Lq, Hq, H, max_len, cur_len);
    return pl.whole ? 0 : (int64_t)pl.wgs * 2 * pl.pitch * (attn::D + 2) * (int64_t)sizeof(float);
}

extern "C" int64_t hn_attn_kv_pages_workspace_size(int64_t B, int64_t Lq, int64_t Hq, int64_t H, int64_t max_len,
                                                   int64_t cur_len) {
    if (!pages_shape_ok(B, Lq, Hq, H, max_len, cur_len)) return 0;
    const PagesPlan pl = pages_plan(B, Lq, Hq / H, H, max_len, cur_len);
    return plan_bytes(pl, B, Lq, Hq, H, max_len, cur_len);
}

extern "C" int hn_attn_kv_pages(int fmt, const void* q, const int64_t* qs, int64_t B, int64_t Lq, int64_t Hq,
                                int64_t D, const void* kc, const void* vc, const int64_t* cs, const float* ks,
                                const float* vs, const int64_t* ss, int64_t H, int64_t n_pages, int64_t page,
                                const int32_t* table, int64_t table_stride, int64_t width, const int32_t* lens,
                                int causal, const int32_t* q_start, const void* kcur, const void* vcur, const int64_t* curs, int64_t cur_len,
                                const uint8_t* cur_valid, int64_t cur_valid_stride, float softmax_scale, void* out,
                                const int64_t* os, float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
    HN_REQUIRE(fmt == HN_KV_FP8 || fmt == HN_KV_INT8, HN_E_ARG, "hn_attn_kv_pages: unknown KV format");
    HN_REQUIRE(D == attn::D, HN_E_ARG, "hn_attn_kv_pages: head dim must be 128");
    HN_REQUIRE(page >= 64 && page <= 1024 && (page & (page - 1)) == 0, HN_E_ARG,
               "hn_attn_kv_pages: page must be 64, 128, 256, 512 or 1024");
    HN_REQUIRE(B >= 0 && Lq >= 0 && H > 0 && Hq > 0 && Hq % H == 0 && n_pages >= 0 && width >= 0 && cur_len >= 0,
               HN_E_ARG, "hn_attn_kv_pages: invalid shape");
    HN_REQUIRE(width <= 0x3fffffffLL / page && n_pages <= 0x7fffffffLL && cur_len <= 0x3fffffffLL, HN_E_ARG,
               "hn_attn_kv_pages: too many keys");
    HN_REQUIRE(!causal || cur_len == 0, HN_E_ARG, "hn_attn_kv_pages: a causal call takes no tail");
    HN_REQUIRE(causal || !q_start, HN_E_ARG, "hn_attn_kv_pages: q_start is a causal call's");
    HN_REQUIRE(softmax_scale > 0.0f && softmax_scale <= 3.4028234e38f, HN_E_ARG,
               "hn_attn_kv_pages: softmax_scale must be finite and positive");
    HN_REQUIRE(qs && os && cs && ss && (cur_len == 0 || curs), HN_E_ARG, "hn_attn_kv_pages: null stride array");
    HN_REQUIRE(qs[3] == 1 && os[3] == 1 && cs[3] == 1, HN_E_ARG, "hn_attn_kv_pages: head dim must be contiguous");
    HN_REQUIRE(qs[0] % 8 == 0 && qs[1] % 8 == 0 && qs[2] % 8 == 0 && os[0] % 4 == 0 && os[1] % 4 == 0 && os[2] % 4 == 0,
               HN_E_ARG, "hn_attn_kv_pages: q/out strides misaligned");
    HN_REQUIRE(cs[0] % 16 == 0 && cs[1] % 16 == 0 && cs[2] % 16 == 0 && cs[0] >= 0 && cs[1] >= 0 && cs[2] >= 0 &&
                   ss[0] >= 0 && ss[1] >= 0 && ss[2] >= 0 && cs[1] <= 0x1ffffffLL && ss[1] <= 0x7fffffLL,
               HN_E_ARG, "hn_attn_kv_pages: pool strides must be multiples of 16 bytes");
    HN_REQUIRE(aligned(q, 16) && aligned(out, 8) && aligned(kc, 16) && aligned(vc, 16) && aligned(ks, 4) &&
                   aligned(vs, 4) && aligned(table, 4) && aligned(lens, 4) && aligned(q_start, 4) && aligned(lse, 4),
               HN_E_ARG, "hn_attn_kv_pages: misaligned pointer");
    HN_REQUIRE(table_stride >= 0 && cur_valid_stride >= 0, HN_E_ARG, "hn_attn_kv_pages: negative stride");
    if (cur_len > 0) {
        HN_REQUIRE(kcur && vcur, HN_E_ARG, "hn_attn_kv_pages: null tail pointer");
        HN_REQUIRE(curs[3] == 1 && curs[0] % 8 == 0 && curs[1] % 8 == 0 && curs[2] % 8 == 0 && curs[0] >= 0 &&
                       curs[1] >= 0 && curs[1] <= 0xffffffLL && curs[2] >= 0,
                   HN_E_ARG, "hn_attn_kv_pages: tail strides must be multiples of 8, below 2^24 per token");
        HN_REQUIRE(aligned(kcur, 16) && aligned(vcur, 16), HN_E_ARG, "hn_attn_kv_pages: tail misaligned");
    }
    if (B == 0 || Lq == 0) return HN_OK;
    HN_REQUIRE(q && out && lse && lens, HN_E_ARG, "hn_attn_kv_pages: null pointer");
    HN_REQUIRE(width == 0 || n_pages == 0 || (table && kc && vc && ks && vs), HN_E_ARG, "hn_attn_kv_pages: null pool pointer");
    const int64_t max_len = n_pages ? width * page : 0;
    HN_REQUIRE(pages_shape_ok(B, Lq, Hq, H, max_len, cur_len), HN_E_ARG, "hn_attn_kv_pages: too much work");
    const PagesPlan pl = pages_plan(B, Lq, Hq / H, H, max_len, cur_len);
    const int64_t units = 1 + (max_len + attn::BKV - 1) / attn::BKV + (cur_len + attn::BKV - 1) / attn::BKV;
    HN_REQUIRE(pl.items <= 0x3fffffffLL / units, HN_E_ARG, "hn_attn_kv_pages: too much work for one launch");
    const int64_t need = plan_bytes(pl, B, Lq, Hq, H, max_len, cur_len);
    HN_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned(workspace, 16))), HN_E_ARG,
               "hn_attn_kv_pages: workspace smaller than hn_attn_kv_pages_workspace_size() or misaligned");
    if (const int rc = require_gfx950("hn_attn_kv_pages"); rc != HN_OK) return rc;
    attn::PageParams p = {};
    p.q = (const uint16_t*)q; p.out = (uint16_t*)out; p.lse = lse;
    p.kc = (const uint8_t*)kc; p.vc = (const uint8_t*)vc; p.ks = ks; p.vs = vs;
    p.kcur = (const uint16_t*)kcur; p.vcur = (const uint16_t*)vcur;
    p.uvalid = cur_len > 0 ? cur_valid : nullptr;
    p.uvs = cur_valid_stride;
    p.table = table; p.lens = lens; p.q_start = q_start; p.ts0 = table_stride;
    p.qs0 = qs[0]; p.qs1 = qs[1]; p.qs2 = qs[2];
    p.os0 = os[0]; p.os1 = os[1]; p.os2 = os[2];
    p.cs0 = cs[0]; p.cs1 = cs[1]; p.cs2 = cs[2];
    p.ss0 = ss[0]; p.ss1 = ss[1]; p.ss2 = ss[2];
    if (max_len == 0) {  // no pool: what the kernels' empty loads are based on is a query's first 256 bytes
        p.kc = p.vc = (const uint8_t*)q;
        p.ks = p.vs = (const float*)q;
        p.cs0 = p.cs1 = p.cs2 = p.ss0 = p.ss1 = p.ss2 = 0;
    }
    if (cur_len > 0) {
        p.us0 = curs[0]; p.us1 = curs[1]; p.us2 = curs[2];
    }
    p.Lq = Lq; p.B = (int)B; p.H = (int)H; p.G = (int)(Hq / H);
    p.rows = (int)(Lq * p.G);
    p.runs = pl.runs;
    p.pages = (int)n_pages;
    p.width = n_pages ? (int)width : 0;
    p.shift = __builtin_ctzll((unsigned long long)page);
    p.cur_len = (int)cur_len;
    p.causal = causal != 0;
    p.scale_log2 = softmax_scale * 1.4426950408889634f;
    if (pl.tiles == 4) return launch_page_tiles(p, fmt, workspace, (hipStream_t)stream);
    p.wgs = pl.wgs;
    p.pitch = pl.pitch;
    if (!pl.whole) {
        p.ws_o = (float*)workspace;
        p.ws_ml = (float*)workspace + (int64_t)pl.wgs * 2 * pl.pitch * attn::D;
    }
    const int64_t grid = pl.whole ? pl.items : pl.wgs;
    p.per_xcd = (int)((grid + 7) / 8);
    const unsigned blocks = 8u * (unsigned)p.per_xcd;
    const hipStream_t st = (hipStream_t)stream;
    if (pl.tiles) {
        attn::Params t = {};
        t.kc = p.kc; t.vc = p.vc; t.ks = p.ks; t.vs = p.vs;
        t.cs0 = p.cs0; t.cs1 = p.cs1; t.cs2 = p.cs2;
        t.ss0 = p.ss0; t.ss1 = p.ss1; t.ss2 = p.ss2;
        t.uvalid = p.uvalid; t.uvs = p.uvs; t.us1 = p.us1;
        if (fmt == HN_KV_FP8) launch_tiles<HN_KV_FP8>(p, t, blocks, st);
        else launch_tiles<HN_KV_INT8>(p, t, blocks, st);
        if (const int rc = check_launch("hn_attn_kv_pages"); rc != HN_OK) return rc;
        return join_pages<attn::BKV>(pl, p, attn::TILE_ROWS, st);
    }
    const bool sv = ss[1] == 1 && ss[0] % 4 == 0 && ss[2] % 4 == 0 && aligned(p.vs, 16);
    if (fmt == HN_KV_FP8) launch_few<HN_KV_FP8>(pl, sv, p, blocks, st);
    else launch_few<HN_KV_INT8>(pl, sv, p, blocks, st);
    if (const int rc = check_launch("hn_attn_kv_pages"); rc != HN_OK || pl.whole) return rc;
    return join_pages<attn::UNIT>(pl, p, 16 * pl.rb, st);
}
