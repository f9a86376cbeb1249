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

// The page of token `pos` of sequence b, or -1.
HN_DEVICE int page_of(const Pool& p, int64_t b, uint32_t pos) {
    const uint32_t i = pos >> p.shift;
    if (i >= (uint32_t)p.width) return -1;
    const int e = p.table[b * p.ts0 + i];
    return (uint32_t)e < (uint32_t)p.pages ? e : -1;
}

// ---------------------------------------------------------------------------
// Quantize-on-write. A row is one (token, head) vector of 128 values: 16 lanes x 8. A
// workgroup's unit is 64 rows, 2^tsh tokens x 64 / 2^tsh heads of one sequence, four
// rows in flight per 16-lane group. HBM bound: 256 bytes read and 132 written a row.
constexpr int UNIT = 64;

struct WriteArgs {
    const uint16_t* x[2];
    uint8_t* q[2];
    float* s[2];
    Pool pool;
    int64_t xs0, xs1, xs2;
    const int32_t* start;
    const int32_t* counts;   // null: L new tokens in every sequence
    int32_t L, H, tsh;
    int32_t ttiles, htiles, units;
    int32_t token_fast;      // rows of a unit are enumerated token by token (tokens lie closer than heads)
    const int32_t* status;
};

struct Row {
    int b, t, h;
    bool there;  // a new token of the sequence
};

HN_DEVICE Row unit_row(const WriteArgs& a, int unit, int r) {
    Row w;
    const int ht = unit % a.htiles, x = unit / a.htiles, tt = x % a.ttiles;
    w.b = x / a.ttiles;
    const int hsh = 6 - a.tsh;
    const int tl = a.token_fast ? r & ((1 << a.tsh) - 1) : r >> hsh, hl = a.token_fast ? r >> a.tsh : r & ((1 << hsh) - 1);
    w.t = (tt << a.tsh) + tl;
    w.h = (ht << hsh) + hl;
    w.there = w.t < a.L && w.h < a.H && (!a.counts || w.t < a.counts[w.b]);
    return w;
}

HN_DEVICE uint4 row_values(const WriteArgs& a, int sel, const Row& w, int lane16) {
    return *reinterpret_cast<const uint4*>(a.x[sel] + w.b * a.xs0 + w.t * a.xs1 + w.h * a.xs2 + lane16 * 8);
}

__global__ void pages_clear_kernel(int32_t* status) {
    if (threadIdx.x == 0) *status = 0;
}

// Sets *status where a new token's value is NaN or Inf (its bf16 exponent is all ones).
__global__ __launch_bounds__(256) void pages_check_kernel(WriteArgs a, int32_t* status) {
    const int lane16 = threadIdx.x & 15, g = threadIdx.x >> 4, sel = blockIdx.y;
    uint32_t bad = 0u;
    for (int unit = blockIdx.x; unit < a.units; unit += gridDim.x) {
        uint4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const Row w = unit_row(a, unit, g + 16 * k);
            v[k] = make_uint4(0u, 0u, 0u, 0u);
            if (w.there) v[k] = row_values(a, sel, w, lane16);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t w[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                bad |= (uint32_t)((w[j] & 0x7f80u) == 0x7f80u) | (uint32_t)((w[j] & 0x7f800000u) == 0x7f800000u);
        }
    }
    if (__any(bad != 0u) && (threadIdx.x & 63) == 0) *status = 1;
}

template <int FMT>
__global__ __launch_bounds__(256) void pages_write_kernel(WriteArgs a) {
    if (a.status != nullptr && *a.status != 0) return;  // refused: nothing is written
    const int lane16 = threadIdx.x & 15, g = threadIdx.x >> 4, sel = blockIdx.y;
    for (int unit = blockIdx.x; unit < a.units; unit += gridDim.x) {
        uint4 v[4];
        Row w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            w[k] = unit_row(a, unit, g + 16 * k);
            if (w[k].there) v[k] = row_values(a, sel, w[k], lane16);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (!w[k].there) continue;
            const int first = a.start[w[k].b];
            const uint32_t pos = (uint32_t)first + (uint32_t)w[k].t;
            const int page = first < 0 ? -1 : page_of(a.pool, w[k].b, pos);
            const uint32_t x[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
            float f[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f[2 * j] = bf16_lo(x[j]);
                f[2 * j + 1] = bf16_hi(x[j]);
            }
            float amax = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(f[j]));
            amax = group_max<16>(amax);
            const float s = amax > 0.0f ? amax / (FMT == HN_KV_FP8 ? kE4M3Max : 127.0f) : 1.0f;
            if (page < 0) continue;
            const int64_t slot = pos & ((1u << a.pool.shift) - 1u);
            *reinterpret_cast<uint2*>(a.q[sel] + page * a.pool.qs0 + slot * a.pool.qs1 + w[k].h * a.pool.qs2 + lane16 * 8) =
                codes8<FMT == HN_KV_FP8>(f, Quot(s));
            if (lane16 == 0) a.s[sel][page * a.pool.ss0 + slot * a.pool.ss1 + w[k].h * a.pool.ss2] = s;
        }
    }
}

// ---------------------------------------------------------------------------
// A sequence decoded: y[b, t, h] = bf16(code * scale), zeros past its length. 16 lanes a
// row, four rows in flight. HBM bound: 132 bytes read and 256 written a row.
struct ReadArgs {
    const uint8_t* q;
    const float* s;
    uint16_t* y;
    Pool pool;
    const int32_t* lens;
    int32_t L, H;
    int64_t rows;  // B L H
};

template <int FMT>
__global__ __launch_bounds__(256) void pages_read_kernel(ReadArgs a) {
    const int lane16 = threadIdx.x & 15, g = threadIdx.x >> 4;
    const uint32_t per = (uint32_t)a.L * (uint32_t)a.H;
    for (int64_t r0 = (int64_t)blockIdx.x * UNIT; r0 < a.rows; r0 += (int64_t)gridDim.x * UNIT) {
        uint2 c[4];
        float s[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t row = r0 + 16 * k + g;
            c[k] = make_uint2(0u, 0u);
            s[k] = 0.0f;
            if (row >= a.rows) continue;
            const int64_t b = row / per;
            const uint32_t in = (uint32_t)(row - b * per), t = in / (uint32_t)a.H, h = in - t * (uint32_t)a.H;
            if ((int)t >= a.lens[b]) continue;
            const int page = page_of(a.pool, b, t);
            if (page < 0) continue;
            const int64_t slot = t & ((1u << a.pool.shift) - 1u);
            c[k] = *reinterpret_cast<const uint2*>(a.q + page * a.pool.qs0 + slot * a.pool.qs1 + h * a.pool.qs2 + lane16 * 8);
            s[k] = a.s[page * a.pool.ss0 + slot * a.pool.ss1 + h * a.pool.ss2];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t row = r0 + 16 * k + g;
            if (row >= a.rows) continue;
            const uint32_t cw[2] = {c[k].x, c[k].y};
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t b0 = (cw[j >> 1] >> (16 * (j & 1))) & 0xffu, b1 = (cw[j >> 1] >> (16 * (j & 1) + 8)) & 0xffu;
                const float v0 = FMT == HN_KV_FP8 ? e4m3_decode(b0) : (float)(int8_t)b0;
                const float v1 = FMT == HN_KV_FP8 ? e4m3_decode(b1) : (float)(int8_t)b1;
                o[j] = f32x2_to_bf16x2(v0 * s[k], v1 * s[k]);
            }
            *reinterpret_cast<uint4*>(a.y + row * 128 + lane16 * 8) = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
}

// ---------------------------------------------------------------------------
// Pages copied, every layer in one launch. The pairs travel in the kernel's arguments,
// so that a copy needs no upload and can be captured; longer lists take several
// launches. A page is one run of bytes in each of the four arrays, moved in pieces of
// 16 KB a workgroup. HBM bound.
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
        if ((int)(threadIdx.x + 256 * k) * 16 < bytes) v[k] = src[threadIdx.x + 256 * k];
#pragma unroll
    for (int k = 0; k < PIECE / 4096; ++k)
        if ((int)(threadIdx.x + 256 * k) * 16 < bytes) dst[threadIdx.x + 256 * k] = v[k];
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

extern "C" int hn_kv_pages_write(int fmt, const void* k, const void* v, const int64_t* xs, int64_t B, int64_t L,
                                 int64_t H, int64_t D, void* kc, void* vc, const int64_t* cs, float* ks, float* vs,
                                 const int64_t* ss, int64_t n_pages, int64_t page, const int32_t* table,
                                 int64_t table_stride, int64_t width, const int32_t* start, const int32_t* counts,
                                 int32_t* status, void* stream) {
    const char* who = "hn_kv_pages_write";
    HN_REQUIRE(fmt == HN_KV_FP8 || fmt == HN_KV_INT8, HN_E_ARG, "hn_kv_pages_write: unknown KV format");
    HN_REQUIRE(D == 128, HN_E_ARG, "hn_kv_pages_write: head dim must be 128");
    HN_REQUIRE(B >= 0 && L >= 0 && H > 0 && B <= 0x7fffffffLL && L <= 0x7fffffffLL && H <= 0x7fffffffLL, HN_E_ARG,
               "hn_kv_pages_write: invalid shape");
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
    if (const int rc = require_gfx950(who); rc != HN_OK) return rc;
    const hipStream_t st = (hipStream_t)stream;
    if (status) pages::pages_clear_kernel<<<1, 64, 0, st>>>(status);
    if (none) return check_launch(who);
    a.x[0] = (const uint16_t*)k; a.x[1] = (const uint16_t*)v;
    a.q[0] = (uint8_t*)kc; a.q[1] = (uint8_t*)vc;
    a.s[0] = ks; a.s[1] = vs;
    a.xs0 = xs[0]; a.xs1 = xs[1]; a.xs2 = xs[2];
    a.start = start; a.counts = counts;
    a.L = (int32_t)L; a.H = (int32_t)H;
    a.token_fast = xs[1] < xs[2];
    a.tsh = 0;
    while (a.tsh < 4 && (1 << a.tsh) < L) ++a.tsh;
    a.ttiles = (int32_t)((L - 1) / (1 << a.tsh) + 1);
    a.htiles = (int32_t)((H - 1) / (pages::UNIT >> a.tsh) + 1);
    HN_REQUIRE(B * a.ttiles <= 0x7fffffffLL / a.htiles, HN_E_ARG, "hn_kv_pages_write: too many rows");
    a.units = (int32_t)(B * a.ttiles * a.htiles);
    a.status = status;
    const dim3 grid((unsigned)stream_grid(a.units, 8), 2);
    if (status) pages::pages_check_kernel<<<grid, 256, 0, st>>>(a, status);
    if (fmt == HN_KV_FP8) pages::pages_write_kernel<HN_KV_FP8><<<grid, 256, 0, st>>>(a);
    else pages::pages_write_kernel<HN_KV_INT8><<<grid, 256, 0, st>>>(a);
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
    HN_REQUIRE(L <= 0x7fffffffLL / H && B <= 0x7fffffffLL, HN_E_ARG, "hn_kv_pages_read: too many rows per sequence");
    if (const int rc = require_gfx950(who); rc != HN_OK) return rc;
    a.q = (const uint8_t*)kc; a.s = ks; a.y = (uint16_t*)y;
    a.lens = lens;
    a.L = (int32_t)L; a.H = (int32_t)H;
    a.rows = B * L * H;
    const unsigned grid = (unsigned)stream_grid((a.rows + pages::UNIT - 1) / pages::UNIT, 16);
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
    int64_t most = 0x7fffffffLL / per_pair;
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
