// Attention over a paged cache: what attn_pages.hip (few rows of queries) and
// attn_blocks.hip (tiles of 128 rows) share.
#pragma once
#include "attn_tiles.h"

namespace hn {
namespace attn {

struct PageParams {
    const uint16_t* q;
    const uint8_t* kc;
    const uint8_t* vc;
    const float* ks;
    const float* vs;
    const uint16_t* kcur;
    const uint16_t* vcur;
    const uint8_t* uvalid;   // null: every tail key is valid
    uint16_t* out;
    float* lse;              // [B, H G, Lq]
    const int32_t* table;
    const int32_t* lens;
    const int32_t* q_start;  // causal: each sequence's first query's token; null: its last Lq tokens are the queries
    int64_t ts0, uvs;
    int64_t qs0, qs1, qs2;
    int64_t cs0, cs1, cs2;   // page, token, head
    int64_t ss0, ss1, ss2;
    int64_t us0, us1, us2;
    int64_t os0, os1, os2;
    int64_t Lq;
    int B, H, G;
    int rows;                // Lq G: row r of a cached head is query r / G, head r % G of its group
    int runs;                // ceil(rows / rows of a workgroup)
    int pages, width, shift; // pool, table row, page = 1 << shift
    int cur_len;
    int causal;
    float scale_log2;
    int wgs;                 // workgroups that the units of all items are dealt out to
    int per_xcd;             // ceil(workgroups / 8)
    int pitch;               // rows of a partial result
    float* ws_o;             // [workgroup][2][pitch][D] unnormalised
    float* ws_ml;            // [workgroup][2][pitch][2]
};

// Integers read by scalar loads: the address is the same in every lane, and no kernel
// that runs at the time writes them.
typedef const __attribute__((address_space(4))) int32_t* ScalarInts;
HN_DEVICE ScalarInts scalar_ints(const int32_t* p) { return (ScalarInts)p; }

// Cached tokens of sequence b that the table can name.
HN_DEVICE int seq_len(const int32_t* lens, int64_t b, int width, int shift) {
    const int n = lens[b], most = width << shift;
    return n < 0 ? 0 : n < most ? n : most;
}

// Causal rows: query i sees tokens below seen_before + i, and below the sequence's length.
template <class P>
HN_DEVICE int seen_before(const P& p, int64_t b, int len) {
    const int first = p.q_start ? __builtin_amdgcn_readfirstlane(p.q_start[b]) : len - (int)p.Lq;
    return (first < len ? first : len) + 1;
}

}  // namespace attn

// The 128-row tile kernel over pages: its workspace, and its launch for the arguments that
// hn_attn_kv_pages has checked.
int64_t page_tiles_workspace(int64_t B, int64_t Lq, int64_t Hq, int64_t H, int64_t max_len, int64_t cur_len);
int launch_page_tiles(const attn::PageParams& p, int fmt, void* workspace, hipStream_t stream);

}  // namespace hn
