// The quantized KV cache in pages (gfx950): new tokens quantized into the pages of
// their sequences, pages copied over the layers, and a paged sequence decoded.
//
// A pool holds `pages` pages of `page` = 1 << shift tokens; token t of sequence b is
// row t & (page - 1) of page table[b, t >> shift]. A table entry outside the pool
// names no page: what would be written there is dropped, what would be read is absent.
// Codes and scales are those of kv_quantize_kernel (quant.hip), bit for bit.
#include "hn_capi_internal.h"
#include "hn_common.h"

namespace hn {
namespace pages {

struct Pool {  // of one of K, V, or of both (same strides)
    int64_t qs0, qs1, qs2;  // codes: page, token, head
    int64_t ss0, ss1, ss2;  // scales
    const int32_t* table;
    int64_t ts0;
    int32_t pages, width, shift;
};

// Loads and stores of what is not read again soon: they pass the caches by. Only where an
// instruction covers whole lines (copy: 61 -> 48 us for eight pages of 40 layers, 259 ->
// 237 for 60; decode with half lines an instruction 94 -> 128).
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
HN_DEVICE void store_once(uint4* p, const uint4& v) {
    __builtin_nontemporal_store((u32x4){v.x, v.y, v.z, v.w}, reinterpret_cast<u32x4*>(p));
}
HN_DEVICE uint4 load_once(const uint4* p) {
    const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
    return make_uint4(v.x, v.y, v.z, v.w);
}

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef const __attribute__((address_space(4))) int32_t* ScalarInts;  // read by scalar loads: no kernel writes them meanwhile

// ---------------------------------------------------------------------------
// Rows are (token, head) vectors of 128 values, 8 lanes x 16 values each. A workgroup's
// tile is 128 rows of one sequence: 2^tsh tokens x 128 / 2^tsh heads, four rows to a lane
// group, their loads in flight together. A tile's tokens lie in two pages at most, whose
// numbers are scalars: with 8 values a lane and the rows' places worked out one by one, the
// instructions were the bound (10800 tokens x 24 heads of two sequences: write 107 us,
// decode 106).
constexpr int TILE = 128;

struct Tiles {
    int32_t L, H, B, tsh;
    int32_t parts;           // tiles of the same tokens: of their heads (write: of K and V of each)
    int32_t token_fast;      // rows are enumerated token by token (tokens lie closer than heads)
};

// A workgroup's tile: the parts of a token range, then the next range, then the next
// sequence; `back`: from the last one on.
struct Place {
    int t0, part;
};

HN_DEVICE Place tile_place(const Tiles& a, bool back) {
    const int x = back ? gridDim.x - 1 - blockIdx.x : blockIdx.x, tt = (uint32_t)x / (uint32_t)a.parts;
    return {tt << a.tsh, x - tt * a.parts};
}

struct Row {
    int t, h;
    bool there;
};

// Row g + 32 k of the tile, g = thread / 8.
HN_DEVICE Row tile_row(const Tiles& a, int t0, int htile, int k, int last) {
    const int r = (threadIdx.x >> 3) + 32 * k, hsh = 7 - a.tsh;
    const int tl = a.token_fast ? r & ((1 << a.tsh) - 1) : r >> hsh, hl = a.token_fast ? r >> a.tsh : r & ((1 << hsh) - 1);
    Row w;
    w.t = t0 + tl;
    w.h = (htile << hsh) + hl;
    w.there = w.t < last && w.h < a.H;
    return w;
}

// The pages of a tile whose first token has position `pos`: of its table entry, and of the
// next one; -1: none.
struct TilePages {
    uint32_t entry;
    int first, next;
};

HN_DEVICE int page_at(const Pool& p, int64_t b, uint32_t entry) {
    if (entry >= (uint32_t)p.width) return -1;
    const int e = ((ScalarInts)(p.table + b * p.ts0))[entry];
    return (uint32_t)e < (uint32_t)p.pages ? e : -1;
}

HN_DEVICE TilePages tile_pages(const Pool& p, int64_t b, uint32_t pos, int tsh) {
    TilePages t;
    t.entry = pos >> p.shift;
    t.first = page_at(p, b, t.entry);
    t.next = ((pos + (1u << tsh) - 1u) >> p.shift) != t.entry ? page_at(p, b, t.entry + 1) : -1;
    return t;
}

HN_DEVICE int page_of(const Pool& p, const TilePages& t, uint32_t pos) {
    return (pos >> p.shift) == t.entry ? t.first : t.next;
}

// Quantize-on-write: s = amax |x| / 448 (127), code = round(x / s). HBM bound: 256 bytes
// read and 132 written a row, and the values a second time by the check that comes before
// (nothing is written where one is not finite). Two sequences of 10800 tokens x 24 heads
// (265 MB of values, 137 MB written): check 45 us (5.9 TB/s), write 68 (5.9).
struct WriteArgs {
    const uint16_t* x[2];
    uint8_t* q[2];
    float* s[2];
    Pool pool;
    int64_t xs0, xs1, xs2;
    const int32_t* start;
    const int32_t* counts;   // null: L new tokens in every sequence
    Tiles tiles;
    float recip;             // not 0: a row's scale is amax times this
    int32_t* status;         // not null: the values are checked, and nothing is written where one is not finite
    uint8_t* flags;          // workspace: a byte of every workgroup of the check
};

HN_DEVICE int new_tokens(const WriteArgs& a, int b) {
    const int n = a.counts ? ((ScalarInts)a.counts)[b] : a.tiles.L;
    return n < a.tiles.L ? n : a.tiles.L;
}

struct Values {
    uint4 a, b;
};

HN_DEVICE Values row_values(const WriteArgs& a, int sel, int b, const Row& w) {
    const uint16_t* x = a.x[sel] + b * a.xs0 + w.t * a.xs1 + w.h * a.xs2 + 16 * (threadIdx.x & 7);
    return {reinterpret_cast<const uint4*>(x)[0], reinterpret_cast<const uint4*>(x)[1]};
}

HN_DEVICE float max8(float v) {  // over the 8 lanes of an aligned group
    v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0xB1, 0xf, 0xf, true)));
    v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x4E, 0xf, 0xf, true)));
    return fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x141, 0xf, 0xf, true)));
}

// The largest magnitudes' bits, of the words' low and high halves.
HN_DEVICE u16x2 largest(u16x2 top, const Values& v) {
    const uint32_t w[8] = {v.a.x, v.a.y, v.a.z, v.a.w, v.b.x, v.b.y, v.b.z, v.b.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w[j] & 0x7fff7fffu));
    return top;
}

__global__ void pages_clear_kernel(int32_t* status) {
    if (threadIdx.x == 0) *status = 0;
}

// Where the check's verdict lies. Up to FLAGS workgroups leave a byte each, which all
// workgroups of the write look at, 16 to a thread; more of them set the status, which a
// launch of its own has cleared (three sequences of up to 777 tokens x 24 heads, 882
// workgroups: kernels 4.7 + 5.3 + 10.7 us by the status, 6.0 + 9.7 by flags; calls 25.7 us
// and 24.3).
enum Check { NONE, ALONE, BY_FLAGS, BY_STATUS };
constexpr int FLAGS = 4096;

// Looks for a new token's value that is NaN or Inf: the largest magnitude's bits of either
// half of the words are then 0x7f80 or more.
template <Check CHECK>
__global__ __launch_bounds__(256) void pages_check_kernel(WriteArgs a) {
    const Place at = tile_place(a.tiles, false);
    const int sel = at.part & 1;
    bool bad = false;
    for (int b = blockIdx.y; b < a.tiles.B; b += gridDim.y) {
        const int last = new_tokens(a, b);
        if (at.t0 >= last) continue;
        Values v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const Row w = tile_row(a.tiles, at.t0, at.part >> 1, k, last);
            v[k] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
            if (w.there) v[k] = row_values(a, sel, b, w);
        }
        u16x2 top = {0, 0};
#pragma unroll
        for (int k = 0; k < 4; ++k) top = largest(top, v[k]);
        bad |= top[0] >= 0x7f80u || top[1] >= 0x7f80u;
    }
    if constexpr (CHECK == BY_STATUS) {
        if (__any(bad) && (threadIdx.x & 63) == 0) *a.status = 1;
    } else {
        const bool any = __syncthreads_or(bad);
        const uint32_t id = blockIdx.y * gridDim.x + blockIdx.x, n = gridDim.x * gridDim.y;
        if (threadIdx.x == 0) a.flags[id] = any;
        if (id == n - 1 && threadIdx.x > 0 && threadIdx.x <= (-n & 15u)) a.flags[id + threadIdx.x] = 0;  // to whole 16
    }
}

// Whether every new value of K and V is finite, looked at by this workgroup alone.
HN_DEVICE bool all_finite(const WriteArgs& a) {
    const uint32_t per = (uint32_t)a.tiles.L * (uint32_t)a.tiles.H, rows = (uint32_t)a.tiles.B * per;
    u16x2 top = {0, 0};
    for (uint32_t r0 = threadIdx.x >> 3; r0 < rows; r0 += 512) {
        Values v[4][2];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t r = r0 + 128 * k, b = r / per, in = r - b * per, t = in / (uint32_t)a.tiles.H;
            const Row w{(int)t, (int)(in - t * (uint32_t)a.tiles.H), r < rows && (!a.counts || (int)t < a.counts[b])};
#pragma unroll
            for (int sel = 0; sel < 2; ++sel) {
                v[k][sel] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
                if (w.there) v[k][sel] = row_values(a, sel, (int)b, w);
            }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) top = largest(top, v[k >> 1][k & 1]);
    }
    return !__syncthreads_or(top[0] >= 0x7f80u || top[1] >= 0x7f80u);
}

// CHECK ALONE: small writes (up to SMALL bytes of values) are one launch, in which every
// workgroup, 1024 threads then, looks at all values: 64 tokens x 8 heads 7.4 us, where
// three kernels take 7.7 and two launches more (calls on either side of the border: 64 tokens
// 15.4 us, 65, of two launches, 19.9).
constexpr int64_t SMALL = 1 << 18;

template <int FMT, Check CHECK>
__global__ __launch_bounds__(CHECK == ALONE ? 1024 : 256) void pages_write_kernel(WriteArgs a) {
    constexpr int NK = CHECK == ALONE ? 1 : 4;  // rows of the tile to a lane group
    const bool first_wg = blockIdx.x == 0 && blockIdx.y == 0;
    if constexpr (CHECK == ALONE) {
        const bool ok = all_finite(a);
        if (first_wg && threadIdx.x == 0) *a.status = !ok;
        if (!ok) return;
    }
    // (asked for here, looked at before the first store: the values' loads do not wait for it)
    int32_t refused = 0;
    uint4 flags = make_uint4(0u, 0u, 0u, 0u);
    if constexpr (CHECK == BY_STATUS) refused = *(ScalarInts)a.status;
    if constexpr (CHECK == BY_FLAGS)
        if (16 * threadIdx.x < gridDim.x * gridDim.y) flags = reinterpret_cast<const uint4*>(a.flags)[threadIdx.x];
    auto verdict = [&]() {
        if constexpr (CHECK != BY_FLAGS) return refused != 0;
        const bool bad = __syncthreads_or((flags.x | flags.y | flags.z | flags.w) != 0u);
        if (first_wg && threadIdx.x == 0) *a.status = bad;
        return bad;
    };
    // (from the last tile on: what the check has read last may be in a cache yet)
    const Place at = tile_place(a.tiles, true);
    const int sel = at.part & 1, t0 = at.t0;
    for (int b = gridDim.y - 1 - blockIdx.y; b < a.tiles.B; b += gridDim.y) {
        const int last = new_tokens(a, b);
        const int first = ((ScalarInts)a.start)[b];
        if (t0 >= last) {
            if (CHECK == BY_FLAGS && first_wg) verdict();  // (for the status)
            continue;
        }
        Values v[NK];
        Row w[NK];
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            w[k] = tile_row(a.tiles, t0, at.part >> 1, k, last);
            if (w[k].there) v[k] = row_values(a, sel, b, w[k]);
        }
        const uint32_t pos0 = (uint32_t)first + (uint32_t)t0;
        const TilePages pages = tile_pages(a.pool, b, pos0, a.tiles.tsh);
        if (verdict()) return;  // nothing is written
        if (first < 0) continue;
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            const uint32_t pos = pos0 + (uint32_t)(w[k].t - t0);
            const int page = page_of(a.pool, pages, pos);
            if (!w[k].there || page < 0) continue;
            const uint32_t x[8] = {v[k].a.x, v[k].a.y, v[k].a.z, v[k].a.w, v[k].b.x, v[k].b.y, v[k].b.z, v[k].b.w};
            float lo[8], hi[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                lo[2 * j] = bf16_lo(x[j]);
                lo[2 * j + 1] = bf16_hi(x[j]);
                hi[2 * j] = bf16_lo(x[4 + j]);
                hi[2 * j + 1] = bf16_hi(x[4 + j]);
            }
            float amax = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fmaxf(fabsf(lo[j]), fabsf(hi[j])));
            amax = max8(amax);
            const float quot = a.recip != 0.0f ? amax * a.recip : amax / (FMT == HN_KV_FP8 ? kE4M3Max : 127.0f);
            const float s = amax > 0.0f ? quot : 1.0f;
            const Quot d(s);
            const uint2 c0 = codes8<FMT == HN_KV_FP8>(lo, d), c1 = codes8<FMT == HN_KV_FP8>(hi, d);
            const int64_t slot = pos & ((1u << a.pool.shift) - 1u);
            uint8_t* q = a.q[sel] + page * a.pool.qs0 + slot * a.pool.qs1 + w[k].h * a.pool.qs2 + 16 * (threadIdx.x & 7);
            store_once(reinterpret_cast<uint4*>(q), make_uint4(c0.x, c0.y, c1.x, c1.y));
            if ((threadIdx.x & 7) == 0) a.s[sel][page * a.pool.ss0 + slot * a.pool.ss1 + w[k].h * a.pool.ss2] = s;
        }
    }
}

// A sequence decoded: y[b, t, h] = bf16(code * scale), zeros past its length. HBM bound:
// 132 bytes read and 256 written a row (1.03 million rows, 401 MB, 69 us: 5.8 TB/s).
struct ReadArgs {
    const uint8_t* q;
    const float* s;
    uint16_t* y;
    Pool pool;
    const int32_t* lens;
    Tiles tiles;
};

// Two codes (bytes 2 hi, 2 hi + 1 of w) -> bf16(code * s), packed.
template <int FMT>
HN_DEVICE uint32_t held2(uint32_t w, bool hi, float s) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    if (FMT == HN_KV_FP8) {
        const f32x2 f = hi ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, 1.0f, true)
                           : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, 1.0f, false);
        return f32x2_to_bf16x2(f[0] * s, f[1] * s);
    }
    const int sh = hi ? 16 : 0;
    return f32x2_to_bf16x2((float)(int8_t)(w >> sh) * s, (float)(int8_t)(w >> (sh + 8)) * s);
}

template <int FMT>
__global__ __launch_bounds__(256) void pages_read_kernel(ReadArgs a) {
    const Place at = tile_place(a.tiles, false);
    const int t0 = at.t0;
    for (int b = blockIdx.y; b < a.tiles.B; b += gridDim.y) {
        const int len = ((ScalarInts)a.lens)[b];
        const TilePages pages = tile_pages(a.pool, b, (uint32_t)t0, a.tiles.tsh);
        uint2 c[4][2];  // dims 8 lane .. and 64 + 8 lane .. of the row: an instruction stores whole lines
        float s[4];
        Row w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            w[k] = tile_row(a.tiles, t0, at.part, k, a.tiles.L);
            c[k][0] = c[k][1] = make_uint2(0u, 0u);
            s[k] = 0.0f;
            const int page = page_of(a.pool, pages, (uint32_t)w[k].t);
            if (!w[k].there || w[k].t >= len || page < 0) continue;
            const int64_t slot = w[k].t & ((1 << a.pool.shift) - 1);
            const uint8_t* q = a.q + page * a.pool.qs0 + slot * a.pool.qs1 + w[k].h * a.pool.qs2 + 8 * (threadIdx.x & 7);
            c[k][0] = *reinterpret_cast<const uint2*>(q);
            c[k][1] = *reinterpret_cast<const uint2*>(q + 64);
            s[k] = a.s[page * a.pool.ss0 + slot * a.pool.ss1 + w[k].h * a.pool.ss2];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (!w[k].there) continue;
            uint4* y = reinterpret_cast<uint4*>(a.y + (((int64_t)b * a.tiles.L + w[k].t) * a.tiles.H + w[k].h) * 128 +
                                                8 * (threadIdx.x & 7));
#pragma unroll
            for (int e = 0; e < 2; ++e)
                store_once(y + 8 * e, make_uint4(held2<FMT>(c[k][e].x, false, s[k]), held2<FMT>(c[k][e].x, true, s[k]),
                                                 held2<FMT>(c[k][e].y, false, s[k]), held2<FMT>(c[k][e].y, true, s[k])));
        }
    }
}

// ---------------------------------------------------------------------------
// Pages copied, every layer in one launch. The pairs travel in the kernel's arguments,
// so that a copy needs no upload and can be captured; longer lists take several
// launches. A page is one run of bytes in each of the four arrays, moved in pieces of
// 16 KB a workgroup, all loads of a thread in flight. HBM bound: 260 MB in 48 us, 1.3 GB in
// 237 (5.4 to 5.5 TB/s; 2 GiB copied in such pieces reach 5.9, in pieces of 4 KB 6.5, by
// torch 4.96).
constexpr int MAX_PAIRS = 240;
constexpr int PIECE = 16384;

struct CopyArgs {
    uint8_t* base[4];      // K and V codes, K and V scales
    int64_t layer[4];      // bytes from layer to layer
    int64_t page[4];       // bytes from page to page
    int32_t size[4];       // bytes of a page
    int32_t piece0[5];     // pieces of a page's arrays before array i; [4]: all
    int32_t layers, n;
    int32_t src[MAX_PAIRS], dst[MAX_PAIRS];
};
static_assert(sizeof(CopyArgs) <= 4096, "kernel arguments");

__global__ __launch_bounds__(256) void pages_copy_kernel(CopyArgs a) {
    const int all = a.piece0[4];
    int x = blockIdx.x;
    const int piece = x % all;
    x /= all;
    const int pair = x % a.n, layer = x / a.n;
    const int i = (piece >= a.piece0[1]) + (piece >= a.piece0[2]) + (piece >= a.piece0[3]);
    const int64_t at = (int64_t)(piece - a.piece0[i]) * PIECE;
    const int64_t left = a.size[i] - at;
    const int bytes = left < PIECE ? (int)left : PIECE;
    uint8_t* const base = a.base[i] + layer * a.layer[i] + at;
    const uint4* src = reinterpret_cast<const uint4*>(base + a.src[pair] * a.page[i]);
    uint4* dst = reinterpret_cast<uint4*>(base + a.dst[pair] * a.page[i]);
    uint4 v[PIECE / 4096];
#pragma unroll
    for (int k = 0; k < PIECE / 4096; ++k)
        if ((int)(threadIdx.x + 256 * k) * 16 < bytes) v[k] = load_once(src + threadIdx.x + 256 * k);
#pragma unroll
    for (int k = 0; k < PIECE / 4096; ++k)
        if ((int)(threadIdx.x + 256 * k) * 16 < bytes) store_once(dst + threadIdx.x + 256 * k, v[k]);
}

}  // namespace pages
}  // namespace hn

using namespace hn;

// ---------------------------------------------------------------------------
// C ABI

static int pool_args(const char* who, const int64_t* cs, const int64_t* ss, int64_t pages_, int64_t page,
                     const int32_t* table, int64_t table_stride, int64_t width, pages::Pool& p) {
    if (!(page >= 64 && page <= 1024 && (page & (page - 1)) == 0)) {
        set_error("%s: page must be 64, 128, 256, 512 or 1024", who);
        return HN_E_ARG;
    }
    if (pages_ < 0 || pages_ > 0x7fffffffLL || width < 0 || width * page > 0x7fffffffLL || table_stride < 0) {
        set_error("%s: invalid pool or table size", who);
        return HN_E_ARG;
    }
    if (!cs || !ss || cs[3] != 1 || cs[0] % 16 || cs[1] % 16 || cs[2] % 16 || cs[0] < 0 || cs[1] < 0 || cs[2] < 0 ||
        ss[0] < 0 || ss[1] < 0 || ss[2] < 0) {
        set_error("%s: pool strides must be multiples of 16 bytes, the head dim contiguous", who);
        return HN_E_ARG;
    }
    p.qs0 = cs[0]; p.qs1 = cs[1]; p.qs2 = cs[2];
    p.ss0 = ss[0]; p.ss1 = ss[1]; p.ss2 = ss[2];
    p.table = table;
    p.ts0 = table_stride;
    p.pages = (int32_t)pages_;
    p.width = (int32_t)width;
    p.shift = __builtin_ctzll((unsigned long long)page);
    return HN_OK;
}

// Tiles of B x L x H rows of `arrays` arrays: as many tokens as there are, up to 16 (eight
// heads beside them), 32 of up to four heads and 64 of two (two sequences of 46057 tokens x 3
// heads: a write 69 us, 94 by 16 tokens). False: too many for one launch.
static bool tiles_of(int64_t B, int64_t L, int64_t H, int arrays, bool token_fast, pages::Tiles& t, dim3& grid) {
    t.B = (int32_t)B; t.L = (int32_t)L; t.H = (int32_t)H;
    t.token_fast = token_fast;
    int most = 4;  // (6 at most: a tile's tokens lie in two pages)
    while (most < 6 && (pages::TILE >> (most + 1)) >= H) ++most;
    t.tsh = 0;
    while (t.tsh < most && (1 << t.tsh) < L) ++t.tsh;
    const int64_t ranges = (L - 1) / (1 << t.tsh) + 1, parts = ((H - 1) / (pages::TILE >> t.tsh) + 1) * arrays;
    if (parts > 0x7fffffffLL || ranges > 0x7fffffffLL / parts) return false;
    t.parts = (int32_t)parts;
    grid = dim3((unsigned)(ranges * parts), (unsigned)(B < 65535 ? B : 65535));
    return true;
}

static pages::Check check_of(const int32_t* status, int64_t B, int64_t L, int64_t H, dim3 grid) {
    if (!status) return pages::NONE;
    if (L * H <= pages::SMALL / (4 * 128) / B) return pages::ALONE;
    return (int64_t)grid.x * grid.y <= pages::FLAGS ? pages::BY_FLAGS : pages::BY_STATUS;
}

static int64_t flag_bytes(dim3 grid) { return ((int64_t)grid.x * grid.y + 15) / 16 * 16; }

template <int FMT>
static void launch_write(pages::Check check, const pages::WriteArgs& a, dim3 grid, hipStream_t st) {
    using namespace pages;
    if (check == ALONE) {
        pages_write_kernel<FMT, ALONE><<<grid, 1024, 0, st>>>(a);
    } else if (check == NONE) {
        pages_write_kernel<FMT, NONE><<<grid, 256, 0, st>>>(a);
    } else if (check == BY_FLAGS) {
        pages_check_kernel<BY_FLAGS><<<grid, 256, 0, st>>>(a);
        pages_write_kernel<FMT, BY_FLAGS><<<grid, 256, 0, st>>>(a);
    } else {
        pages_clear_kernel<<<1, 64, 0, st>>>(a.status);
        pages_check_kernel<BY_STATUS><<<grid, 256, 0, st>>>(a);
        pages_write_kernel<FMT, BY_STATUS><<<grid, 256, 0, st>>>(a);
    }
}

static bool write_shape_ok(int64_t B, int64_t L, int64_t H) {
    return B >= 0 && L >= 0 && H > 0 && B <= 0x7fffffffLL && L <= 0x7fffffffLL && H <= 0x7fffffffLL;
}

extern "C" int64_t hn_kv_pages_write_workspace_size(int64_t B, int64_t L, int64_t H) {
    pages::Tiles tiles;
    dim3 grid;
    if (!write_shape_ok(B, L, H) || B == 0 || L == 0 || !tiles_of(B, L, H, 2, false, tiles, grid)) return 0;
    const int32_t checked = 0;
    return check_of(&checked, B, L, H, grid) == pages::BY_FLAGS ? flag_bytes(grid) : 0;
}

extern "C" int hn_kv_pages_write(int fmt, const void* k, const void* v, const int64_t* xs, int64_t B, int64_t L,
                                 int64_t H, int64_t D, void* kc, void* vc, const int64_t* cs, float* ks, float* vs,
                                 const int64_t* ss, int64_t n_pages, int64_t page, const int32_t* table,
                                 int64_t table_stride, int64_t width, const int32_t* start, const int32_t* counts,
                                 int scale_mode, int32_t* status, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
    const char* who = "hn_kv_pages_write";
    HN_REQUIRE(fmt == HN_KV_FP8 || fmt == HN_KV_INT8, HN_E_ARG, "hn_kv_pages_write: unknown KV format");
    HN_REQUIRE(scale_mode == HN_SCALE_ZERO_ONE || scale_mode == HN_SCALE_RECIPROCAL, HN_E_ARG,
               "hn_kv_pages_write: unknown scale mode");
    HN_REQUIRE(D == 128, HN_E_ARG, "hn_kv_pages_write: head dim must be 128");
    HN_REQUIRE(write_shape_ok(B, L, H), HN_E_ARG, "hn_kv_pages_write: invalid shape");
    pages::WriteArgs a = {};
    if (const int rc = pool_args(who, cs, ss, n_pages, page, table, table_stride, width, a.pool); rc != HN_OK) return rc;
    HN_REQUIRE(xs && xs[3] == 1 && xs[0] % 8 == 0 && xs[1] % 8 == 0 && xs[2] % 8 == 0, HN_E_ARG,
               "hn_kv_pages_write: value strides must be multiples of 8, the head dim contiguous");
    HN_REQUIRE(aligned(k, 16) && aligned(v, 16) && aligned(kc, 16) && aligned(vc, 16) && aligned(ks, 4) &&
                   aligned(vs, 4) && aligned(table, 4) && aligned(start, 4) && aligned(counts, 4) && aligned(status, 4),
               HN_E_ARG, "hn_kv_pages_write: misaligned pointer");
    const bool none = B == 0 || L == 0;
    if (none && !status) return HN_OK;
    HN_REQUIRE(none || (k && v && start && (n_pages == 0 || (kc && vc && ks && vs)) && (width == 0 || table)), HN_E_ARG,
               "hn_kv_pages_write: null pointer");
    if (none) {
        if (const int rc = require_gfx950(who); rc != HN_OK) return rc;
        pages::pages_clear_kernel<<<1, 64, 0, (hipStream_t)stream>>>(status);
        return check_launch(who);
    }
    a.x[0] = (const uint16_t*)k; a.x[1] = (const uint16_t*)v;
    a.q[0] = (uint8_t*)kc; a.q[1] = (uint8_t*)vc;
    a.s[0] = ks; a.s[1] = vs;
    a.xs0 = xs[0]; a.xs1 = xs[1]; a.xs2 = xs[2];
    a.start = start; a.counts = counts;
    if (scale_mode == HN_SCALE_RECIPROCAL) a.recip = 1.0f / (fmt == HN_KV_FP8 ? kE4M3Max : 127.0f);
    dim3 grid;
    HN_REQUIRE(tiles_of(B, L, H, 2, xs[1] < xs[2], a.tiles, grid), HN_E_ARG, "hn_kv_pages_write: too many rows");
    a.status = status;
    a.flags = (uint8_t*)workspace;
    const pages::Check check = check_of(status, B, L, H, grid);
    HN_REQUIRE(check != pages::BY_FLAGS || (workspace && aligned(workspace, 16) && workspace_bytes >= flag_bytes(grid)),
               HN_E_ARG, "hn_kv_pages_write: workspace smaller than hn_kv_pages_write_workspace_size() or misaligned");
    if (const int rc = require_gfx950(who); rc != HN_OK) return rc;
    if (fmt == HN_KV_FP8) launch_write<HN_KV_FP8>(check, a, grid, (hipStream_t)stream);
    else launch_write<HN_KV_INT8>(check, a, grid, (hipStream_t)stream);
    return check_launch(who);
}

extern "C" int hn_kv_pages_read(int fmt, const void* kc, const int64_t* cs, const float* ks, const int64_t* ss,
                                int64_t n_pages, int64_t page, const int32_t* table, int64_t table_stride,
                                int64_t width, const int32_t* lens, int64_t B, int64_t L, int64_t H, int64_t D,
                                void* y, void* stream) {
    const char* who = "hn_kv_pages_read";
    HN_REQUIRE(fmt == HN_KV_FP8 || fmt == HN_KV_INT8, HN_E_ARG, "hn_kv_pages_read: unknown KV format");
    HN_REQUIRE(D == 128, HN_E_ARG, "hn_kv_pages_read: head dim must be 128");
    HN_REQUIRE(B >= 0 && L >= 0 && H > 0, HN_E_ARG, "hn_kv_pages_read: invalid shape");
    pages::ReadArgs a = {};
    if (const int rc = pool_args(who, cs, ss, n_pages, page, table, table_stride, width, a.pool); rc != HN_OK) return rc;
    HN_REQUIRE(aligned(kc, 16) && aligned(ks, 4) && aligned(y, 16) && aligned(table, 4) && aligned(lens, 4), HN_E_ARG,
               "hn_kv_pages_read: misaligned pointer");
    if (B == 0 || L == 0) return HN_OK;
    HN_REQUIRE(y && lens && (width == 0 || table) && (n_pages == 0 || (kc && ks)), HN_E_ARG,
               "hn_kv_pages_read: null pointer");
    HN_REQUIRE(B <= 0x7fffffffLL && L <= 0x7fffffffLL && H <= 0x7fffffffLL, HN_E_ARG, "hn_kv_pages_read: too many rows");
    if (const int rc = require_gfx950(who); rc != HN_OK) return rc;
    a.q = (const uint8_t*)kc; a.s = ks; a.y = (uint16_t*)y;
    a.lens = lens;
    dim3 grid;
    HN_REQUIRE(tiles_of(B, L, H, 1, false, a.tiles, grid), HN_E_ARG, "hn_kv_pages_read: too many rows");
    if (fmt == HN_KV_FP8) pages::pages_read_kernel<HN_KV_FP8><<<grid, 256, 0, (hipStream_t)stream>>>(a);
    else pages::pages_read_kernel<HN_KV_INT8><<<grid, 256, 0, (hipStream_t)stream>>>(a);
    return check_launch(who);
}

extern "C" int hn_kv_pages_copy(void* const* base, const int64_t* layer_stride, const int64_t* page_stride,
                                const int64_t* page_bytes, int64_t layers, int64_t n_pages, const int32_t* src,
                                const int32_t* dst, int64_t n, void* stream) {
    const char* who = "hn_kv_pages_copy";
    HN_REQUIRE(layers >= 0 && n >= 0 && n_pages >= 0, HN_E_ARG, "hn_kv_pages_copy: invalid shape");
    if (layers == 0 || n == 0) return HN_OK;
    HN_REQUIRE(base && layer_stride && page_stride && page_bytes && src && dst, HN_E_ARG, "hn_kv_pages_copy: null pointer");
    HN_REQUIRE(layers <= 0xffff, HN_E_ARG, "hn_kv_pages_copy: too many layers");
    pages::CopyArgs a = {};
    a.layers = (int32_t)layers;
    for (int i = 0; i < 4; ++i) {
        HN_REQUIRE(base[i] && aligned(base[i], 16) && layer_stride[i] % 16 == 0 && page_stride[i] % 16 == 0 &&
                       page_bytes[i] % 16 == 0,
                   HN_E_ARG, "hn_kv_pages_copy: arrays, strides and sizes must be multiples of 16 bytes");
        HN_REQUIRE(page_bytes[i] > 0 && page_bytes[i] <= (1 << 28) && page_stride[i] >= page_bytes[i], HN_E_ARG,
                   "hn_kv_pages_copy: pages overlap");
        a.base[i] = (uint8_t*)base[i];
        a.layer[i] = layer_stride[i];
        a.page[i] = page_stride[i];
        a.size[i] = (int32_t)page_bytes[i];
        a.piece0[i + 1] = a.piece0[i] + (int32_t)((page_bytes[i] + pages::PIECE - 1) / pages::PIECE);
    }
    for (int64_t i = 0; i < n; ++i)
        HN_REQUIRE(src[i] >= 0 && src[i] < n_pages && dst[i] >= 0 && dst[i] < n_pages, HN_E_ARG,
                   "hn_kv_pages_copy: a page outside the pool");
    if (const int rc = require_gfx950(who); rc != HN_OK) return rc;
    const int64_t per_pair = (int64_t)a.piece0[4] * layers;
    int64_t most = 0xffffffLL / per_pair;  // (a grid has fewer than 2^32 threads)
    HN_REQUIRE(most > 0, HN_E_ARG, "hn_kv_pages_copy: a page of all layers is too large");
    most = most < pages::MAX_PAIRS ? most : pages::MAX_PAIRS;
    for (int64_t i0 = 0; i0 < n; i0 += most) {
        a.n = (int32_t)(n - i0 < most ? n - i0 : most);
        for (int j = 0; j < a.n; ++j) {
            a.src[j] = src[i0 + j];
            a.dst[j] = dst[i0 + j];
        }
        pages::pages_copy_kernel<<<(unsigned)(per_pair * a.n), 256, 0, (hipStream_t)stream>>>(a);
        if (const int rc = check_launch(who); rc != HN_OK) return rc;
    }
    return HN_OK;
}
