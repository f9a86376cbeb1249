// Key/value tiles of the attention kernels over the quantized KV cache (gfx950):
// the tile layout in LDS, its loads from the cache and from the bf16 tail, the
// dequantizing writes, and the two software-pipelined steps of a half tile
// (S^T = K Q^T beside the probabilities, O^T += V^T P^T beside the next tile's
// write). attn_fp8kv.hip describes the scheme; attn_blocks.hip runs the same
// steps over a list of cache blocks.
#pragma once
#include "hn_capi_internal.h"
#include "hn_common.h"

namespace hn {
namespace attn {

constexpr int D = 128;
constexpr int BKV = 64;            // keys per tile
constexpr int QW = 32;             // queries per wave
constexpr int KROW = D * 2 + 16;   // K tile row: 128 bf16 + 16 B pad (bank spread)
// V^T tile: 128 dim rows of 64 fp16 keys (128 B) padded to 144 B = 9 16-byte
// units, so 16 consecutive rows at one column fall in 16 different bank
// groups (9 is odd). Column unit c of a row holds the 8 keys 16 (c / 2) +
// 4 (c % 2) + {0..3} and + 8 + {0..3}: the keys lane half c % 2 feeds to the
// PV MFMA for 16-key slice c / 2.
constexpr int VTROW = 144;
constexpr int K_BYTES = BKV * KROW;
constexpr int VT_BYTES = D * VTROW;
// After K and V^T, each stage holds the tile's 64-bit key-validity word (bit
// j: key j of the tile exists and is valid), written only by the MASK
// instantiation.
constexpr int MASK_OFF = K_BYTES + VT_BYTES;
constexpr int STAGE = K_BYTES + VT_BYTES + 16;
constexpr uint64_t ALL_KEYS = ~0ull;
// Per-key scales of a tile in flight ([0, 64) K, [64, 128) V), two buffers.
constexpr int SB_FLOATS = 2 * BKV;
// K/V stages in LDS: three for the 8-wave shape (one workgroup per CU), so
// that a tile is written two tiles ahead of its use and one barrier per tile
// suffices; two for the 4-wave shape, whose two workgroups per CU could not
// hold three each.
template <int NW>
constexpr int stages() { return NW == 8 ? 3 : 2; }
template <int NW>
constexpr int smem_bytes() { return stages<NW>() * STAGE + 2 * SB_FLOATS * 4; }

// Workgroup shape for NW (4 or 8) waves.
template <int NW>
struct Shape {
    static_assert(NW == 4 || NW == 8, "4 or 8 waves");
    static constexpr int NT = 64 * NW;   // threads
    static constexpr int BQ = QW * NW;   // queries
    static constexpr int KU = 512 / NT;  // 16-code K units per thread (64 keys x 8 units)
    static constexpr int VD = 2048 / NT; // V dims per thread (64 keys x 128 dims, 4-key quads)
};

struct Params {
    const uint16_t* q;
    const uint8_t* kc;
    const uint8_t* vc;
    const float* ks;
    const float* vs;
    const uint16_t* kcur;
    const uint16_t* vcur;
    uint16_t* out;
    // Key-validity bytes (MASK instantiation; null = every key valid): cache
    // keys kvalid[b * kvs + t], tail keys uvalid[b * uvs + j].
    const uint8_t* kvalid;
    const uint8_t* uvalid;
    int64_t kvs, uvs;
    int64_t qs0, qs1, qs2;
    int64_t cs0, cs1, cs2;   // cs0 == 0 (and ss0 == 0): one cache slot read by every batch
    int64_t ss0, ss1, ss2;
    int64_t us0, us1, us2;
    int64_t os0, os1, os2;
    int64_t Lq, H, kv_len, cur_len, q_pos0, chunk;
    float scale_log2;  // softmax_scale * log2(e)
    int fmt;
    int q_tiles;       // ceil(Lq / BQ)
    int splits;        // key-range splits per (batch, head, query tile)
    int work;          // B * H * q_tiles * splits
    int per_xcd;       // ceil(work / 8)
    float* ws_o;       // splits > 1: unnormalized O, [split][B][H][Lq][D] fp32
    float* ws_ml;      // splits > 1: running max and sum, [split][B][H][Lq][2]
};

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// ---------------------------------------------------------------------------
// Dequantization to the reference's bf16 values.

// Two codes (bytes 2 hi, 2 hi + 1 of w) -> their exact fp32 values. The gfx950
// conversion is used with a unit scale only: its scale operand applies just
// the exponent of the fp32 value.
template <int FMT>
HN_DEVICE f32x2 codes2_f32(uint32_t w, bool hi) {
    if (FMT == HN_KV_FP8)
        return hi ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, 1.0f, true)
                  : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, 1.0f, false);
    const uint32_t sh = hi ? 16 : 0;
    f32x2 r;
    r[0] = (float)(int8_t)((w >> sh) & 0xffu);
    r[1] = (float)(int8_t)((w >> (sh + 8)) & 0xffu);
    return r;
}

// bf16 bits of fp32 a and b, packed (a low), round to nearest even.
HN_DEVICE uint32_t pack_bf16(float a, float b) {
    const f32x2 f = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2));
}

// fp16 bits of fp32 a and b, packed (a low), round to nearest even.
HN_DEVICE uint32_t pack_f16(float a, float b) {
    const f32x2 f = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, f16x2));
}

// fp16 bits of bf16(a), bf16(b): the reference's bf16 dequantized values held
// as fp16 operands of the PV MFMA. Each value is rounded as the high half of a
// pair whose low half is 0, which is the fp32 form of its bf16 value as it
// stands: 3 instructions for two values, where rounding them as one pair and
// taking it apart again costs 4. Exact for bf16 values in fp16's normal range;
// the pack rounds toward zero, so magnitudes past 65504 saturate.
HN_DEVICE uint32_t pack_f16_of_bf16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(__uint_as_float(pack_bf16(0.0f, a)),
                                                                   __uint_as_float(pack_bf16(0.0f, b))));
}

// ---------------------------------------------------------------------------
// Tile loads and LDS writes.
//
// K: thread t owns units i < KU: key k_key(t) + NT / 8 i, 16 dims at 16 k_unit(t).
// In each wave, lane bits 0-1 give the unit's low bits, bit 2 the key's low
// bit, bit 3 the unit's high bit and bits 4-5 the key's high bits: 16 lanes
// cover two whole key rows (256 contiguous bytes of the cache), and the
// 16-byte LDS writes of any 8 consecutive lanes (two keys, rows 272 B apart)
// fall in 8 different 16-byte bank groups -- a 16-byte LDS write is served 8
// lanes at a time over 128 bytes of banks, so one key's 8 units 32 B apart
// would pair up.
// V^T: thread t (wave w, lane λ) owns key quad qd = λ % 16 (keys quad_key(qd, j),
// j < 4: the 8-byte half qd % 2 of column unit qd / 2) and the VD dims VD dg ..
// VD dg + VD - 1 (v_group). Per 8-byte LDS write a 32-lane group covers 2 dim
// groups 8 rows apart x 16 quads, whose bank pairs (18 row + qd) mod 32 are all
// distinct (row pitch 144 B, 18 x 8 = 16 mod 32); per global load each wave
// reads 16 keys x 4 VD contiguous bytes.
// Scales: threads 0-63 load the K scale of key t, threads 64-127 the V scale
// of key t - 64, into the tile's scale buffer.
// Validity (MASK): threads 128-191 (wave 2) load the validity byte of key
// t - 128; the wave's ballot is the tile's validity word.

// Key (within the tile, for i = 0) and unit (16-code run of the key) of
// thread t's K unit.
HN_DEVICE uint32_t k_key(uint32_t t) { return 8u * (t >> 6) + 2u * ((t >> 4) & 3u) + ((t >> 2) & 1u); }
HN_DEVICE uint32_t k_unit(uint32_t t) { return (t & 3u) + 4u * ((t >> 3) & 1u); }

// Key (0..63) of entry j (0..3) of quad qd.
HN_DEVICE int quad_key(int qd, int j) {
    return 16 * (qd >> 2) + 4 * ((qd >> 1) & 1) + 8 * (qd & 1) + j;
}

// Dim group of this thread's V^T quad: lanes 0-31 and 32-63 of a wave take
// groups whose first rows are 8 apart.
template <int NW>
HN_DEVICE int v_group_of(int tid) {
    const int w = tid >> 6, hh = (tid & 63) >> 4;
    if constexpr (NW == 4) return 4 * w + hh;                       // 8 dims per group
    else return 4 * w + 2 * (hh & 1) + (hh >> 1);                   // 4 dims per group
}
template <int NW>
HN_DEVICE int v_group() { return v_group_of<NW>(threadIdx.x); }

// Registers holding one cache tile between its global load and its LDS
// write (issued about one tile ahead).
template <int NW>
struct CacheRegs {
    uint4 k[Shape<NW>::KU];
    uint32_t v[4][Shape<NW>::VD / 4];  // VD codes (dims VD dg ..) of quad key j
    float s;                           // one per-key scale (threads < 128)
    uint32_t mk;                       // MASK: validity of key t - 128 (wave 2)
};

// A cache tile's loads are buffer loads: per tile one scalar descriptor per
// array (base = the tile's first key; size = the tile's bytes, so rows past
// the tile's key count read as zeros -- they are masked out of the softmax --
// with no per-lane clamp), and per lane a fixed 32-bit offset inside the
// tile, computed once (LaneOffs).
constexpr int BUF_FLAGS = 0x00020000;  // raw (stride 0) buffer, 32-bit dwords

struct TileBase {
    __amdgpu_buffer_rsrc_t k, v, ks, vs;
    const uint8_t* mk;  // validity bytes of the tile's keys, or null (all valid)
};

HN_DEVICE __amdgpu_buffer_rsrc_t tile_rsrc(const void* base, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes, BUF_FLAGS);
}

// count = 0 gives empty descriptors: every load through them reads zeros and
// touches no memory (the loop issues its prefetch loads unconditionally, so
// that their order, and with it every wait on them, is the same on all paths).
HN_DEVICE TileBase tile_base(const Params& p, int64_t b, int64_t h, int64_t first, int count) {
    TileBase tb;
    const int64_t c = b * p.cs0 + first * p.cs1 + h * p.cs2;
    const int64_t s = b * p.ss0 + first * p.ss1 + h * p.ss2;
    const int64_t cb = count > 0 ? (int64_t)(count - 1) * p.cs1 + D : 0;  // codes of keys 0 .. count - 1
    const int64_t sb = count > 0 ? ((int64_t)(count - 1) * p.ss1 + 1) * 4 : 0;
    tb.k = tile_rsrc(p.kc + c, cb);
    tb.v = tile_rsrc(p.vc + c, cb);
    tb.ks = tile_rsrc(p.ks + s, sb);
    tb.vs = tile_rsrc(p.vs + s, sb);
    tb.mk = p.kvalid ? p.kvalid + b * p.kvs + first : nullptr;
    return tb;
}

// This thread's byte offsets inside a tile: K units (key u / 8, 16 codes at
// 16 (u % 8)), the VD codes of its V^T quad keys, and its per-key scale
// (threads < 128: K scales for threads 0-63, V for 64-127).
template <int NW>
struct LaneOffs {
    uint32_t k[Shape<NW>::KU];
    uint32_t v[4];
    uint32_t s;
};

template <int NW>
HN_DEVICE LaneOffs<NW> lane_offsets(const Params& p) {
    LaneOffs<NW> o;
    const uint32_t t = threadIdx.x;
#pragma unroll
    for (int i = 0; i < Shape<NW>::KU; ++i)
        o.k[i] = (k_key(t) + (uint32_t)(Shape<NW>::NT / 8) * i) * (uint32_t)p.cs1 + k_unit(t) * 16u;
    const int qd = t & 15, dg = v_group<NW>();
#pragma unroll
    for (int j = 0; j < 4; ++j) o.v[j] = (uint32_t)quad_key(qd, j) * (uint32_t)p.cs1 + (uint32_t)(Shape<NW>::VD * dg);
    o.s = (t & 63u) * (uint32_t)p.ss1 * 4u;
    return o;
}

// `co` / `so`: a tile's byte offset inside descriptors that start before it
// (the steady loop's span descriptors), added to every lane's code / scale
// offset; `mk0` the tile's first key in the span's validity bytes; 0 with
// per-tile descriptors.
template <int NW, bool MASK>
HN_DEVICE void load_k(const LaneOffs<NW>& lo, CacheRegs<NW>& r, const TileBase& tb, int count, uint32_t co = 0,
                      uint32_t so = 0, int64_t mk0 = 0) {
    const uint32_t t = threadIdx.x;
    // Wave 0 reads the K scales, wave 1 the V scales. The wave index goes
    // through readfirstlane so that the descriptor choice is a scalar one (a
    // per-lane choice of descriptor would be a loop over its distinct values).
    // The scale load is issued before the codes: its consumer (the scale
    // buffer write) then waits for it alone.
    const uint32_t wv = __builtin_amdgcn_readfirstlane(t >> 6);
    if (wv < 2u) {
        const __amdgpu_buffer_rsrc_t sr = wv == 0u ? tb.ks : tb.vs;
        r.s = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(sr, lo.s + so, 0, 0));
    }
#pragma unroll
    for (int i = 0; i < Shape<NW>::KU; ++i)
        r.k[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(tb.k, lo.k[i] + co, 0, 0));
    if constexpr (MASK) {
        if ((t >> 6) == 2u) {
            const uint32_t j = t & 63u;
            r.mk = (int)j < count ? (tb.mk ? (uint32_t)tb.mk[mk0 + j] : 1u) : 0u;
        }
    }
}

// The validity word of a cache tile, from the bytes wave 2 loaded with its
// codes, into the stage (MASK only). Called with the tile's K write.
template <int NW, bool MASK>
HN_DEVICE void store_mask(const CacheRegs<NW>& r, uint8_t* st) {
    if constexpr (MASK) {
        if ((threadIdx.x >> 6) == 2) {
            const uint64_t bits = __ballot(r.mk != 0u);
            if ((threadIdx.x & 63) == 0) *reinterpret_cast<uint64_t*>(st + MASK_OFF) = bits;
        }
    }
}

// The validity word of the tile in stage st (ALL_KEYS without MASK). Every
// lane reads the same 8 bytes; the word is made wave-uniform.
template <bool MASK>
HN_DEVICE uint64_t tile_mask(const uint8_t* st) {
    if constexpr (!MASK) return ALL_KEYS;
    const uint64_t w = *reinterpret_cast<const uint64_t*>(st + MASK_OFF);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)w);
    const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(w >> 32));
    return ((uint64_t)hi << 32) | lo;
}

template <int NW>
HN_DEVICE void load_v(const LaneOffs<NW>& lo, CacheRegs<NW>& r, const TileBase& tb, uint32_t co = 0) {
    constexpr int VD = Shape<NW>::VD;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (VD == 8) {
            const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(tb.v, lo.v[j] + co, 0, 0));
            r.v[j][0] = x.x;
            r.v[j][1] = x.y;
        } else {
            r.v[j][0] = __builtin_amdgcn_raw_buffer_load_b32(tb.v, lo.v[j] + co, 0, 0);
        }
    }
}

HN_DEVICE uint32_t word(const uint4& c, int q) { return q == 0 ? c.x : q == 1 ? c.y : q == 2 ? c.z : c.w; }

// Dequantized K write, part i (0..7): the thread's codes 2 KU i .. +2 KU - 1
// (unit code / 16) into bf16 dwords of kd; each completed run of 8 codes is
// one 16-byte write (every second part with 2 units, every fourth with 1).
template <int FMT, int NW>
HN_DEVICE void store_k_part(const CacheRegs<NW>& r, uint8_t* st, int i, const float (&ks)[Shape<NW>::KU],
                            uint32_t (&kd)[4]) {
    constexpr int CP = 2 * Shape<NW>::KU;  // codes per part
    const int code0 = CP * i, un = code0 >> 4, c = code0 & 15;
#pragma unroll
    for (int c2 = 0; c2 < CP / 2; ++c2) {
        const int cc = c + 2 * c2;
        const f32x2 a = codes2_f32<FMT>(word(r.k[un], cc >> 2), (cc & 2) != 0);
        kd[(cc >> 1) & 3] = pack_bf16(a[0] * ks[un], a[1] * ks[un]);
    }
    if (((c + CP) & 7) == 0) {
        const uint32_t key = k_key(threadIdx.x) + (Shape<NW>::NT / 8) * un;
        *reinterpret_cast<uint4*>(st + key * KROW + k_unit(threadIdx.x) * 32 + ((c + CP - 8) >> 3) * 16) =
            make_uint4(kd[0], kd[1], kd[2], kd[3]);
    }
}

// The K scales of the thread's units, from the tile's scale buffer.
template <int NW>
HN_DEVICE void k_scales(const float* sb, float (&ks)[Shape<NW>::KU]) {
#pragma unroll
    for (int i = 0; i < Shape<NW>::KU; ++i) ks[i] = sb[k_key(threadIdx.x) + (Shape<NW>::NT / 8) * i];
}

// Dequantized V^T write, part i (0..7): quad key j = i / 2, dims VD/2 (i % 2)
// .. + VD/2 - 1 of the thread's VD; keys (0, 1) and (2, 3) pair into dwords
// of fp16-held bf16 values (vd[2 d + pair], dim d), and parts 6 and 7 write
// the two halves of the dims (8 bytes = 4 keys each).
// `vc` holds the thread's codes (as CacheRegs::v), `vt` is the V^T tile.
template <int FMT, int NW>
HN_DEVICE void store_v_part(const uint32_t (&vc)[4][Shape<NW>::VD / 4], uint8_t* vt, int i, const float4& vs,
                            float (&vp)[Shape<NW>::VD], uint32_t (&vd)[2 * Shape<NW>::VD]) {
    constexpr int VD = Shape<NW>::VD, DP = VD / 2;
    const int j = i >> 1, hf = i & 1;
    const float s = j == 0 ? vs.x : j == 1 ? vs.y : j == 2 ? vs.z : vs.w;
    float x[DP];
#pragma unroll
    for (int c2 = 0; c2 < DP / 2; ++c2) {
        const int code = DP * hf + 2 * c2;
        const f32x2 a = codes2_f32<FMT>(vc[j][code >> 2], (code & 2) != 0);
        x[2 * c2] = a[0] * s;
        x[2 * c2 + 1] = a[1] * s;
    }
#pragma unroll
    for (int dd = 0; dd < DP; ++dd) {
        const int d = DP * hf + dd;
        if (j & 1) vd[2 * d + (j >> 1)] = pack_f16_of_bf16(vp[d], x[dd]);
        else vp[d] = x[dd];
    }
    if (j == 3) {
        const int qd = threadIdx.x & 15, dg = v_group<NW>();
#pragma unroll
        for (int dd = 0; dd < DP; ++dd) {
            const int d = DP * hf + dd;
            *reinterpret_cast<uint2*>(vt + (VD * dg + d) * VTROW + 8 * qd) = make_uint2(vd[2 * d], vd[2 * d + 1]);
        }
    }
}

// The V scales of the thread's quad (4 consecutive keys), from the scale buffer.
HN_DEVICE float4 v_scales(const float* sb) {
    const int qd = threadIdx.x & 15;
    return *reinterpret_cast<const float4*>(sb + BKV + quad_key(qd, 0));
}

// Whole-tile write (prologue), scales from the tile's scale buffer.
template <int FMT, int NW, bool MASK>
HN_DEVICE void store_tile(const CacheRegs<NW>& r, uint8_t* st, const float* sb) {
    store_mask<NW, MASK>(r, st);
    float ks[Shape<NW>::KU];
    k_scales<NW>(sb, ks);
    const float4 vs = v_scales(sb);
    uint32_t kd[4];
    float vp[Shape<NW>::VD];
    uint32_t vd[2 * Shape<NW>::VD];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        store_k_part<FMT, NW>(r, st, i, ks, kd);
        store_v_part<FMT, NW>(r.v, st + K_BYTES, i, vs, vp, vd);
    }
}

// Unquantized tail tile (bf16 K/V of the current chunk), written with the
// same thread-to-location mapping as the cache writes (so it cleanly
// replaces what those wrote to the same stage). The loads and the LDS writes
// are separate steps: the tail loops of both shapes, and the 8-wave general
// loop, issue a tail tile's loads ahead into TailRegs, as they do a cache
// tile's; the 4-wave general loop (which holds a cache tile's prefetch beside
// it, near the register limit) loads and writes in one go (copy_tail_k / _v).
template <int NW>
struct TailRegs {
    uint4 k[2 * Shape<NW>::KU];        // unit i: dims 16 u .. + 7 in k[2 i], + 8 .. + 15 in k[2 i + 1]
    uint32_t v[4][Shape<NW>::VD / 2];  // dims VD dg .. + VD - 1 of quad key j (bf16 pairs)
    uint32_t mk;                       // MASK: validity of key t - 128 (wave 2)
};

template <int NW, bool MASK>
HN_DEVICE void load_tail_k(const Params& p, int64_t b, int64_t h, int64_t first, int count, TailRegs<NW>& r) {
    const int t = threadIdx.x;
    if constexpr (MASK) {
        if ((t >> 6) == 2) {
            const int j = t & 63;
            r.mk = j < count ? (p.uvalid ? (uint32_t)p.uvalid[b * p.uvs + first + j] : 1u) : 0u;
        }
    }
#pragma unroll
    for (int i = 0; i < Shape<NW>::KU; ++i) {
        const int key = (int)k_key(t) + (Shape<NW>::NT / 8) * i, unit = (int)k_unit(t);
        const int j = min(key, count - 1);
        const uint16_t* src = p.kcur + b * p.us0 + (first + j) * p.us1 + h * p.us2 + unit * 16;
        r.k[2 * i] = *reinterpret_cast<const uint4*>(src);
        r.k[2 * i + 1] = *reinterpret_cast<const uint4*>(src + 8);
    }
}

template <int NW, bool MASK>
HN_DEVICE void store_tail_mask(const TailRegs<NW>& r, uint8_t* st) {
    if constexpr (MASK) {
        if ((threadIdx.x >> 6) == 2) {
            const uint64_t bits = __ballot(r.mk != 0u);
            if ((threadIdx.x & 63) == 0) *reinterpret_cast<uint64_t*>(st + MASK_OFF) = bits;
        }
    }
}

// 16-byte half `hf` of unit i's 32 bytes.
template <int NW>
HN_DEVICE void store_tail_k_part(const TailRegs<NW>& r, uint8_t* st, int i, int hf) {
    const int key = (int)k_key(threadIdx.x) + (Shape<NW>::NT / 8) * i;
    reinterpret_cast<uint4*>(st + key * KROW + (int)k_unit(threadIdx.x) * 32)[hf] = r.k[2 * i + hf];
}

template <int NW, bool MASK>
HN_DEVICE void store_tail_k(const TailRegs<NW>& r, uint8_t* st) {
    store_tail_mask<NW, MASK>(r, st);
#pragma unroll
    for (int i = 0; i < 2 * Shape<NW>::KU; ++i) store_tail_k_part<NW>(r, st, i >> 1, i & 1);
}

template <int NW>
HN_DEVICE void load_tail_v(const Params& p, int64_t b, int64_t h, int64_t first, int count, TailRegs<NW>& r) {
    constexpr int VD = Shape<NW>::VD;
    const int qd = threadIdx.x & 15, dg = v_group<NW>();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int key = min(quad_key(qd, j), count - 1);
        const uint16_t* src = p.vcur + b * p.us0 + (first + key) * p.us1 + h * p.us2 + VD * dg;
        if constexpr (VD == 8) {
            const uint4 x = *reinterpret_cast<const uint4*>(src);
            r.v[j][0] = x.x; r.v[j][1] = x.y; r.v[j][2] = x.z; r.v[j][3] = x.w;
        } else {
            const uint2 x = *reinterpret_cast<const uint2*>(src);
            r.v[j][0] = x.x; r.v[j][1] = x.y;
        }
    }
}

// V^T holds fp16: the bf16 values converted (exactly, in fp16's range). Part d:
// the thread's dim d, 4 keys.
template <int NW>
HN_DEVICE void store_tail_v_part(const TailRegs<NW>& r, uint8_t* st, int d) {
    constexpr int VD = Shape<NW>::VD;
    const int qd = threadIdx.x & 15, dg = v_group<NW>();
    uint32_t o[2];
#pragma unroll
    for (int pr = 0; pr < 2; ++pr) {
        const uint32_t a = r.v[2 * pr][d >> 1], b = r.v[2 * pr + 1][d >> 1];
        o[pr] = __builtin_bit_cast(uint32_t, (d & 1) ? __builtin_amdgcn_cvt_pkrtz(bf16_hi(a), bf16_hi(b))
                                                     : __builtin_amdgcn_cvt_pkrtz(bf16_lo(a), bf16_lo(b)));
    }
    *reinterpret_cast<uint2*>(st + K_BYTES + (VD * dg + d) * VTROW + 8 * qd) = make_uint2(o[0], o[1]);
}

template <int NW>
HN_DEVICE void store_tail_v(const TailRegs<NW>& r, uint8_t* st) {
#pragma unroll
    for (int d = 0; d < Shape<NW>::VD; ++d) store_tail_v_part<NW>(r, st, d);
}

// Steady tail tiles: loads through descriptors spanning the (batch, head) tail
// rows [0, tail_end), at the tile's byte offset `co` (rows past the end read as
// zeros), with the lane's offsets inside a tile.
template <int NW>
struct TailOffs {
    uint32_t k[Shape<NW>::KU], v[4];
};

template <int NW>
HN_DEVICE TailOffs<NW> tail_offsets(const Params& p) {
    TailOffs<NW> o;
    const uint32_t t = threadIdx.x, pitch = 2 * (uint32_t)p.us1;
#pragma unroll
    for (int i = 0; i < Shape<NW>::KU; ++i)
        o.k[i] = (k_key(t) + (uint32_t)(Shape<NW>::NT / 8) * i) * pitch + k_unit(t) * 32u;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        o.v[j] = (uint32_t)quad_key(t & 15, j) * pitch + (uint32_t)(2 * Shape<NW>::VD * v_group<NW>());
    return o;
}

template <int NW, bool MASK>
HN_DEVICE void load_tail_span_k(const Params& p, int64_t b, const TailOffs<NW>& lo, __amdgpu_buffer_rsrc_t k,
                                uint32_t co, int64_t first, int64_t end, TailRegs<NW>& r) {
    if constexpr (MASK) {
        if ((threadIdx.x >> 6) == 2) {
            const int64_t j = first + (threadIdx.x & 63);
            r.mk = j < end ? (p.uvalid ? (uint32_t)p.uvalid[b * p.uvs + j] : 1u) : 0u;
        }
    }
#pragma unroll
    for (int i = 0; i < Shape<NW>::KU; ++i) {
        r.k[2 * i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(k, lo.k[i] + co, 0, 0));
        r.k[2 * i + 1] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(k, lo.k[i] + co + 16, 0, 0));
    }
}

template <int NW>
HN_DEVICE void load_tail_span_v(const TailOffs<NW>& lo, __amdgpu_buffer_rsrc_t v, uint32_t co, TailRegs<NW>& r) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (Shape<NW>::VD == 8) {
            const uint4 x = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(v, lo.v[j] + co, 0, 0));
            r.v[j][0] = x.x; r.v[j][1] = x.y; r.v[j][2] = x.z; r.v[j][3] = x.w;
        } else {
            const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(v, lo.v[j] + co, 0, 0));
            r.v[j][0] = x.x; r.v[j][1] = x.y;
        }
    }
}

template <int NW, bool MASK>
HN_DEVICE void copy_tail_k(const Params& p, int64_t b, int64_t h, int64_t first, int count, uint8_t* st) {
    TailRegs<NW> r;
    load_tail_k<NW, MASK>(p, b, h, first, count, r);
    store_tail_k<NW, MASK>(r, st);
}

template <int NW>
HN_DEVICE void copy_tail_v(const Params& p, int64_t b, int64_t h, int64_t first, int count, uint8_t* st) {
    TailRegs<NW> r;
    load_tail_v<NW>(p, b, h, first, count, r);
    store_tail_v<NW>(r, st);
}

HN_DEVICE f32x16 mfma_bf16(const bf16x8& a, const bf16x8& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

HN_DEVICE f32x16 mfma_f16(const f16x8& a, const f16x8& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

HN_DEVICE bf16x8 ld_bf16x8(const uint8_t* p) {
    return __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(p));
}

HN_DEVICE f16x8 ld_f16x8(const uint8_t* p) {
    return __builtin_bit_cast(f16x8, *reinterpret_cast<const uint4*>(p));
}

// Max of v over the lane pair (l, l ^ 32), through the LDS crossbar
// (ds_bpermute). gfx950's v_permlane32_swap is not used: in this kernel's
// instruction stream the compiler issues it two wait states after the VALU
// write of its operand, and the swapped values were then stale (the running
// max came out lane-local, which fp16 probabilities turn into overflow).
HN_DEVICE float pair_max(float v) { return fmaxf(v, __shfl_xor(v, 32, 64)); }

// ---------------------------------------------------------------------------
// Half-tile steps. A "half" is one 32-key block kb of a 64-key tile; for it
// the wave holds S^T as one f32x16 (register v: key 32 kb + 8 (v/4) + 4 half
// + v%4, query = this lane's column).

// S^T block kb of the tile in stage st: 8 MFMAs over the 128 dims (prologue).
HN_DEVICE f32x16 s_block(const uint8_t* ka, const bf16x8 (&qf)[8]) {
    f32x16 acc;
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[v] = 0.0f;
#pragma unroll
    for (int sl = 0; sl < 8; ++sl) acc = mfma_bf16(ld_bf16x8(ka + 32 * sl), qf[sl], acc);
    return acc;
}

// Running state of this lane's query: m, the reference point of the
// probabilities in log2 units (-inf before any visible key); nm = -m (0 while
// m = -inf); l, this lane's share of the softmax denominator.
struct Run {
    float m, nm, l;
};

// m may lag the true running max by up to REBASE_SLACK: the probabilities
// 2^(s c - m) then stay <= 2^REBASE_SLACK, far inside fp16's range, and O, l
// and m stay consistent (both are relative to m), so the softmax is the same
// for any such m.
constexpr float REBASE_SLACK = 8.0f;

// Max of a raw S^T block over this lane's 16 keys of the query (the pair
// lane holds the other 16; rebase exchanges the two only when it acts).
HN_DEVICE float raw_max(const f32x16& s) {
    float mx = s[0];
#pragma unroll
    for (int v = 1; v < 16; ++v) mx = fmaxf(mx, s[v]);
    return mx;
}

// Partial tiles: keys j >= lim of the tile, and keys whose bit of the tile's
// validity word mw is clear, are masked to -inf; returns the new max.
HN_DEVICE float mask_raw(f32x16& u, int kb, int half, int lim, uint64_t mw) {
    const uint32_t bits = (uint32_t)(mw >> (kb * 32 + 4 * half));
    float mx = -INFINITY;
#pragma unroll
    for (int v = 0; v < 16; ++v) {
        const int j = kb * 32 + 8 * (v >> 2) + 4 * half + (v & 3);
        if (j >= lim || !((bits >> (8 * (v >> 2) + (v & 3))) & 1u)) u[v] = -INFINITY;
        mx = fmaxf(mx, u[v]);
    }
    return mx;
}

// A block whose keys' validity is the same for every query: bit j of w is key j
// of the block. The two halves of the wave hold different keys, so register v's
// lane mask is one bit of w for lanes 0-31 and another for lanes 32-63, made by
// scalar instructions: one select per logit, where mask_raw's per-lane bit and
// limit tests take about four more. Returns the new max. 7712 masked queries
// over 14 912 keys with 2 % holes: 1.980 -> 1.970 ms.
HN_DEVICE float mask_word(f32x16& u, uint32_t w) {
#pragma unroll
    for (int v = 0; v < 16; ++v) {
        const int j = 8 * (v >> 2) + (v & 3);
        const uint64_t lo = (w >> j) & 1u ? 0xffffffffull : 0ull, hi = (w >> (j + 4)) & 1u ? 0xffffffffull : 0ull;
        u[v] = __builtin_amdgcn_inverse_ballot_w64(hi << 32 | lo) ? u[v] : -INFINITY;
    }
    return raw_max(u);
}

// Before a block's probabilities, with the lane's raw block max mx (its
// logit max in log2 units is mx * c, c = softmax_scale * log2 e > 0): taken,
// wave-uniformly, only when some lane's logit max passes m + REBASE_SLACK
// (always when a lane sees its first visible key, m = -inf). Then m moves to
// the pair's exact max (an LDS-crossbar exchange with lane ^ 32), and O and l
// are rescaled by 2^(m_old - m_new).
HN_DEVICE void rebase(float mx, float c, Run& run, f32x16 (&o)[4]) {
    if (!__any(mx * c > run.m + REBASE_SLACK)) return;
    const float mnew = fmaxf(run.m, pair_max(mx) * c);
    const float alpha = run.m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(run.m - mnew);
    run.m = mnew;
    run.nm = mnew == -INFINITY ? 0.0f : -mnew;  // m = -inf: every s is -inf (masked)
    run.l *= alpha;
    if (__any(alpha != 1.0f)) {
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int v = 0; v < 16; ++v) o[db][v] *= alpha;
    }
}

// Ties values to this point of the instruction stream: the empty asm is
// ordered with the sched_barrier that ends a slot, so the arithmetic feeding
// it cannot drift into later slots (pure operations are otherwise placed
// freely before the machine scheduler sees the barrier).
template <typename A, typename B, typename C>
HN_DEVICE void pin(A& a, B& b, C& c) {
    asm volatile("" : "+v"(a), "+v"(b), "+v"(c));
}
template <typename A, typename B>
HN_DEVICE void pin(A& a, B& b) {
    asm volatile("" : "+v"(a), "+v"(b));
}
template <typename A>
HN_DEVICE void pin(A& a) {
    asm volatile("" : "+v"(a));
}

// ---------------------------------------------------------------------------
// The two software-pipelined steps of a half tile. Each pairs one 8-MFMA chain
// with the independent VALU work of the other chain, spread over 8 slots (one
// MFMA + about 8 VALU instructions, ~32 cycles each) that sched_barrier keeps
// in place: a wave's VALU instructions execute while its own MFMAs occupy the
// matrix core, so the overlap is built into each wave's instruction stream
// rather than left to the other wave on the SIMD. Operand reads from LDS are
// issued two slots ahead.

// Step A: S^T of the next block from the K rows at ka (this lane's row in the
// stage) beside the probabilities of the current block (raw S^T in s):
// p = 2^(s c - m), l += fp16(p), P^T = fp16(p) for the two 16-key slices
// (registers 8t .. 8t+7 hold keys 16 t + 4 half + {0..3} and + 8 + {0..3} of
// the block).
HN_DEVICE f32x16 step_a(const f32x16& s, float c, float nm, float& l, f16x8 (&pf)[2], const uint8_t* ka,
                        const bf16x8 (&qf)[8]) {
    bf16x8 kf[8];
    kf[0] = ld_bf16x8(ka);
    kf[1] = ld_bf16x8(ka + 32);
    f32x16 acc;
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[v] = 0.0f;
    float ls = 0.0f;
    const f16x2 ones = {(_Float16)1.0f, (_Float16)1.0f};
    uint32_t x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (i + 2 < 8) kf[i + 2] = ld_bf16x8(ka + 32 * (i + 2));
        acc = mfma_bf16(kf[i], qf[i], acc);
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * i], c, nm));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * i + 1], c, nm));
        x[i] = pack_f16(p0, p1);
        // l sums the fp16 probabilities the PV MFMA multiplies (v_dot2_f32_f16)
        ls = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, x[i]), ones, ls, false);
        pin(x[i], ls);
        __builtin_amdgcn_sched_barrier(0);
    }
    l += ls;
    pf[0] = __builtin_bit_cast(f16x8, make_uint4(x[0], x[1], x[2], x[3]));
    pf[1] = __builtin_bit_cast(f16x8, make_uint4(x[4], x[5], x[6], x[7]));
    return acc;
}

// Step B: O^T += V^T P^T of block kb (V^T operand reads at va: this lane's
// row and column in the stage) beside the raw max of the next block (s) and,
// in slot i, beside(i). Returns the next block's raw max over this lane's keys.
template <typename F>
HN_DEVICE float step_b_with(const f16x8 (&pf)[2], const uint8_t* va, int kb, f32x16 (&o)[4], const f32x16& s,
                            F beside) {
    // operand i (= 4 tt + db): dim block db, 16-key slice 2 kb + tt
    f16x8 vf[8];
    vf[0] = ld_f16x8(va + 64 * kb);
    vf[1] = ld_f16x8(va + 64 * kb + 32 * VTROW);
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int tt = i >> 2, db = i & 3;
        if (i + 2 < 8) {
            const int i2 = i + 2;
            vf[i2] = ld_f16x8(va + 64 * kb + 32 * (i2 >> 2) + (i2 & 3) * 32 * VTROW);
        }
        o[db] = mfma_f16(vf[i], pf[tt], o[db]);
        mx = fmaxf(mx, fmaxf(s[2 * i], s[2 * i + 1]));
        pin(mx);
        beside(i);
        __builtin_amdgcn_sched_barrier(0);
    }
    return mx;
}

// Step B beside half of the write of the prefetched cache tile (STORE 1: K, 2:
// V^T) to stage nst with the scales of buffer sb.
template <int FMT, int NW, int STORE>
HN_DEVICE float step_b(const f16x8 (&pf)[2], const uint8_t* va, int kb, f32x16 (&o)[4], const f32x16& s,
                       const CacheRegs<NW>& r, uint8_t* nst, const float* sb) {
    float ks[Shape<NW>::KU] = {};
    float4 vs = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (STORE == 1) k_scales<NW>(sb, ks);
    if (STORE == 2) vs = v_scales(sb);
    uint32_t kd[4];
    float vp[Shape<NW>::VD];
    uint32_t vd[2 * Shape<NW>::VD];
    return step_b_with(pf, va, kb, o, s, [&](int i) __attribute__((always_inline)) {
        if (STORE == 1) store_k_part<FMT, NW>(r, nst, i, ks, kd);
        if (STORE == 2) store_v_part<FMT, NW>(r.v, nst + K_BYTES, i, vs, vp, vd);
    });
}

// ---------------------------------------------------------------------------
// The steps of the kernels that return a row's log-sum-exp.

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

// rebase with the running maximum held 2^11 low: probabilities are 2^11 to
// 2^15 where a row's largest is, so that fp16 holds those down to 2^-25 of it in full
// (2^-14 with the largest at 1) and what lies below is off by 2^-36 of it. Over a long
// history many small weights add up to what one large one leaves. (The slack shrinks
// from 2^8 to 2^4: fp16 ends at 2^16.)
constexpr float PROB_LOG2 = 11.0f, PROB_TOP = 15.0f;

HN_DEVICE void rebase_high(float mx, float c, Run& run, f32x16 (&o)[4]) {
    if (!__any(mx * c > run.m + PROB_TOP)) return;
    const float mnew = fmaxf(run.m, pair_max(mx) * c - PROB_LOG2);
    const float alpha = run.m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(run.m - mnew);
    run.m = mnew;
    run.nm = mnew == -INFINITY ? 0.0f : -mnew;  // m = -inf: every s is -inf (masked)
    run.l *= alpha;
    if (__any(alpha != 1.0f)) {
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int v = 0; v < 16; ++v) o[db][v] *= alpha;
    }
}

}  // namespace attn
}  // namespace hn
