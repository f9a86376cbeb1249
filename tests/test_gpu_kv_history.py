"""GPU tests of the long-history operators against plain 64-bit forms: block
bounds, block choice, attention over listed blocks, key mass, eviction.

Tolerances count the roundings on the way (half a step each, relative to the
value: bf16 2^-8, fp16 2^-11, fp32 2^-24):
  * logits are fp32 sums of 128 exact products: off by at most e_s = 128 2^-24
    sum |q k| scale, which moves a probability by that much relative;
  * the exponent's argument |x| <= X is rounded once or twice (X 2^-23), the
    exponential itself is good to 2^-22;
  * fp32 chains of n positive terms are off by at most n 2^-24 relative.
Bounds, chosen indices and moved rows are compared for equality."""
import math

import pytest
import torch

from conftest import pkg_module

pytestmark = pytest.mark.gpu
F64, BF16, INF = torch.float64, torch.bfloat16, float("inf")
D, SCALE = 128, 128 ** -0.5


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _cache(dev, B, cap, H, fmt, g, layout="bshd", gain=1.5):
    """A written cache; "bhsd": stored head by head, "wide": rows of a wider buffer."""
    kvc = pkg_module("fp8_kv_cache")
    make = kvc.make_fp8_kv_block if fmt == "fp8" else kvc.make_int8_kv_block
    if layout == "bshd":
        cache = make(B, cap, H, D, device=dev)
    elif layout == "bhsd":
        cache = {n: t.transpose(1, 2) for n, t in make(B, H, cap, D, device=dev).items()}
    else:
        cache = {n: t[:, :, 1:1 + H, :] for n, t in make(B, cap, H + 2, D, device=dev).items()}
    if cap:
        k = (torch.randn(B, cap, H, D, device=dev, generator=g) * gain).to(BF16)
        v = (torch.randn(B, cap, H, D, device=dev, generator=g) * gain).to(BF16)
        kvc.quantize_kv_pair_into(cache, k, v, 0)
    return cache


def _held(cache, key):
    return (cache[key].float() * cache[key + "_scale"]).to(BF16).to(F64)


def _poison(cache, tokens):
    """NaN scales and codes in rows that no call may look at (tokens: bool [B, cap])."""
    for key in ("k", "v"):
        cache[key + "_scale"][tokens] = float("nan")
        codes = cache[key]
        raw = codes.view(torch.uint8)
        raw[tokens] = 0x7f


# --------------------------------------------------------------------------
# bounds

def _bounds_reference(old, cache, start, end, block, valid):
    out = old.to(F64).clone()
    k = _held(cache, "k")
    if start == end:
        return out
    for j in range(start // block, -(-end // block)):
        t0, t1 = j * block, min((j + 1) * block, end)
        x = k[:, t0:t1]
        ok = torch.ones(x.shape[:2], dtype=torch.bool, device=x.device) if valid is None else \
            valid[:, t0:t1].bool().expand(x.shape[0], -1)
        ok = ok[:, :, None, None]
        out[:, j, :, 0] = torch.where(ok, x, INF).amin(1)
        out[:, j, :, 1] = torch.where(ok, x, -INF).amax(1)
    return out


@pytest.mark.parametrize("B,cap,H,start,end,block,fmt,layout,holes", [
    (1, 64, 1, 0, 64, 64, "fp8", "bshd", 0),
    (2, 300, 3, 0, 300, 64, "fp8", "bshd", 0.3),       # a ragged last block
    (1, 300, 3, 130, 131, 64, "int8", "bshd", 0),      # one appended token: its whole block
    (2, 1000, 5, 64, 700, 128, "int8", "bhsd", 0.1),
    (1, 1100, 2, 1, 1025, 1024, "fp8", "wide", 0.5),   # one block and one token of the next
    (3, 70, 24, 69, 70, 64, "fp8", "wide", 0),
    (1, 520, 4, 200, 200, 64, "fp8", "bshd", 0),       # nothing written: nothing changes
    (1, 513, 7, 256, 513, 256, "fp8", "bhsd", 0.9),
])
def test_block_bounds(dev, B, cap, H, start, end, block, fmt, layout, holes):
    print(f"case bounds B={B} cap={cap} H={H} [{start},{end}) block={block} {fmt} {layout}", flush=True)
    hist = pkg_module("kv_history")
    g = _gen(dev, cap + end)
    cache = _cache(dev, B, cap, H, fmt, g, layout)
    valid = (torch.rand(B, cap, device=dev, generator=g) >= holes) if holes else None
    if holes == 0.5:
        valid[:, :1024] = False                        # a block without a valid token
    bounds = hist.make_block_bounds(cache, block=block)
    assert torch.isinf(bounds.float()).all()
    bounds[:, 0] = 7.0                                 # (rows outside the call's blocks stay)
    ref = _bounds_reference(bounds, cache, start, end, block, valid)
    unread = torch.zeros(B, cap, dtype=torch.bool, device=dev)
    unread[:, end:] = True
    if valid is not None:
        unread |= ~valid
    _poison(cache, unread)
    hist.update_block_bounds(bounds, cache, start, end, block=block, cache_valid=valid)
    assert torch.equal(bounds.to(F64), ref)
    if valid is not None:                              # uint8 masks of wider rows count the same
        again = torch.full_like(bounds, 3.0)
        wide = torch.zeros(B, cap + 9, dtype=torch.uint8, device=dev)
        wide[:, :cap] = valid.to(torch.uint8) * 5
        hist.update_block_bounds(again, cache, start, end, block=block, cache_valid=wide)
        j0, j1 = start // block, -(-end // block)
        assert torch.equal(again[:, j0:j1], bounds[:, j0:j1])


# --------------------------------------------------------------------------
# block choice

def _choose(scores, forced, empty, k):
    """Ascending indices of the k best (forced first, ties to the lowest), -1 behind."""
    order = sorted((j for j in range(len(scores)) if not empty[j]),
                   key=lambda j: (not forced[j], -scores[j] if not forced[j] else 0, j))
    got = sorted(order[:k])
    return got + [-1] * (k - len(got))


def _select_reference(q, bounds, kv_len, top_k, block, q_block, first, last, q_valid):
    """Exact sums (math.fsum), each score rounded once to fp32."""
    import numpy as np
    B, Lq, Hq, _ = q.shape
    H = bounds.shape[2]
    G, n, runs = Hq // H, -(-kv_len // block), -(-Lq // q_block)
    qd = q.to(F64).cpu().numpy()
    bd = bounds.to(F64).cpu().numpy()
    out = []
    for b in range(B):
        bb = b if bounds.shape[0] == B else 0
        for h in range(H):
            for r in range(runs):
                rows = [i for i in range(r * q_block, min((r + 1) * q_block, Lq))
                        if q_valid is None or bool(q_valid[b if q_valid.shape[0] > 1 else 0, i])]
                x = qd[b, rows][:, h * G:(h + 1) * G].reshape(-1, D)
                W = [math.fsum(c) for c in np.minimum(x, 0).T] if len(x) else [0.0] * D
                U = [math.fsum(c) for c in np.maximum(x, 0).T] if len(x) else [0.0] * D
                scores, empty = [], []
                for j in range(n):
                    lo, hi = bd[bb, j, h]
                    empty.append(bool(lo[0] > hi[0]))
                    s = 0.0 if empty[-1] else math.fsum([*(a * c for a, c in zip(W, lo)), *(a * c for a, c in zip(U, hi))])
                    scores.append(float(np.float32(s)))
                forced = [j < first or j >= n - last for j in range(n)]
                out.append(_choose(scores, forced, empty, top_k))
    return torch.tensor(out, dtype=torch.int32).reshape(B, H, runs, top_k)


def _random_bounds(dev, B, n, H, g, gone=0.0, ties=False):
    centre = torch.randn(B, n, H, D, device=dev, generator=g)
    if ties:
        centre = centre[:, :1].expand(-1, n, -1, -1)
    spread = torch.rand(B, 1 if ties else n, H, D, device=dev, generator=g)
    bounds = torch.stack([centre - spread, centre + spread], 3).to(BF16)
    if gone:
        no = torch.rand(B, n, device=dev, generator=g) < gone
        bounds[:, :, :, 0] = torch.where(no[:, :, None, None], INF, bounds[:, :, :, 0])
        bounds[:, :, :, 1] = torch.where(no[:, :, None, None], -INF, bounds[:, :, :, 1])
    return bounds.contiguous()


@pytest.mark.parametrize("B,Lq,Hq,H,kv_len,block,q_block,top_k,first,last,gone,q_holes,slots", [
    (1, 1, 1, 1, 64, 64, 1, 1, 0, 0, 0, 0, 1),
    (1, 1, 8, 2, 5000, 64, 1, 8, 1, 2, 0.2, 0, 1),          # single tokens of grouped heads
    (2, 3, 6, 3, 4100, 128, 1, 40, 0, 1, 0, 0, 2),          # more entries than blocks
    (2, 300, 3, 3, 6411, 64, 128, 16, 4, 4, 0.1, 0.3, 1),   # ragged runs, padded queries, one slot
    (1, 130, 4, 1, 20000, 64, 64, 5, 0, 0, 0, 0, 1),        # two runs and two queries
    (1, 40, 2, 2, 9000, 256, 7, 3, 3, 0, 0, 0, 1),          # only the first blocks
    (1, 700, 2, 2, 12345, 64, 33, 11, 1, 1, 0.05, 0, 1),    # many runs
    (1, 9, 2, 1, 70, 64, 4, 3, 0, 0, 1.0, 0, 1),            # no block with a token
])
def test_select_blocks(dev, B, Lq, Hq, H, kv_len, block, q_block, top_k, first, last, gone, q_holes, slots):
    print(f"case select B={B} Lq={Lq} Hq={Hq}/{H} kv={kv_len} block={block} q_block={q_block} k={top_k}", flush=True)
    hist = pkg_module("kv_history")
    g = _gen(dev, Lq + kv_len)
    n = -(-kv_len // block)
    q = torch.randn(B, Lq, Hq, D, device=dev, generator=g).to(BF16)
    bounds = _random_bounds(dev, slots, n + 2, H, g, gone)
    q_valid = (torch.rand(B, Lq, device=dev, generator=g) >= q_holes) if q_holes else None
    if q_valid is not None:
        q = torch.where(q_valid[:, :, None, None], q, float("nan"))   # what padded rows hold does not matter
    got = hist.select_blocks(q, bounds, kv_len, top_k, block=block, q_block=q_block, keep_first=first, keep_last=last,
                             q_valid=q_valid)
    ref = _select_reference(q, bounds, kv_len, top_k, block, q_block, first, last, q_valid)
    assert got.dtype == torch.int32 and torch.equal(got.cpu(), ref)


def test_select_blocks_ties_and_strides(dev):
    """Equal scores go to the lowest index; strided queries and bounds; no history."""
    hist = pkg_module("kv_history")
    g = _gen(dev, 3)
    q = torch.randn(1, 70, 4, D, device=dev, generator=g).to(BF16)
    bounds = _random_bounds(dev, 1, 600, 2, g, ties=True)
    got = hist.select_blocks(q, bounds, 600 * 64, 20, q_block=32)
    assert torch.equal(got.cpu(), torch.arange(20, dtype=torch.int32).expand(1, 2, 3, 20))
    got = hist.select_blocks(q, bounds, 600 * 64, 20, q_block=32, keep_last=3)
    assert torch.equal(got[0, 0, 0].cpu().long(), torch.tensor([*range(17), 597, 598, 599]))
    bounds = _random_bounds(dev, 2, 50, 2, g)
    wide = torch.zeros(2, 50, 5, 2, D, dtype=BF16, device=dev)
    wide[:, :, 2:4] = bounds
    qt = torch.randn(2, 4, 70, D + 8, device=dev, generator=g).to(BF16)[..., :D].transpose(1, 2)
    got = hist.select_blocks(qt, wide[:, :, 2:4], 50 * 64 - 7, 9, q_block=32)
    assert torch.equal(got.cpu(), _select_reference(qt, bounds, 50 * 64 - 7, 9, 64, 32, 0, 0, None))
    assert (hist.select_blocks(q, bounds[:1], 0, 4) == -1).all()
    assert hist.select_blocks(q[:, :0], bounds[:1], 640, 4).shape == (1, 2, 0, 4)
    # a NaN query: every score is NaN and ranks as -inf, so the lowest indices
    qn = q.clone()
    qn[0, 0, 0, 5] = float("nan")
    assert hist.select_blocks(qn, bounds[:1], 640, 4, q_block=70)[0, 0, 0].tolist() == [0, 1, 2, 3]


# --------------------------------------------------------------------------
# attention over listed blocks

def _attend(q, cache, kv_len, idx, block, q_block, k_cur, v_cur, valid, cur_valid, scale=SCALE):
    """(out, lse, tolerances) in 64 bits."""
    B, Lq, Hq, _ = q.shape
    H = cache["k"].shape[2]
    G = Hq // H
    k, v = _held(cache, "k"), _held(cache, "v")
    dev = q.device
    out = torch.zeros(B, Lq, Hq, D, dtype=F64, device=dev)
    lse = torch.full((B, Hq, Lq), -INF, dtype=F64, device=dev)
    tol_o, tol_l = torch.zeros_like(out), torch.zeros_like(lse)
    lists = None if idx is None else idx.cpu().tolist()
    for b in range(B):
        c = b if k.shape[0] == B else 0
        ok = torch.ones(k.shape[1], dtype=torch.bool, device=dev)
        if valid is not None:
            ok[:valid.shape[1]] = valid[b if valid.shape[0] > 1 else 0].bool()[:k.shape[1]]
        for h in range(H):
            for r in range(-(-Lq // q_block)):
                if lists is None:
                    t = torch.arange(kv_len, device=dev)
                else:
                    names = []
                    for j in lists[b][h][r]:
                        if j < 0:
                            break
                        names.append(j)
                    t = torch.tensor([x for j in names for x in range(j * block, min((j + 1) * block, kv_len))],
                                     dtype=torch.long, device=dev)
                t = t[ok[t]]
                keys, vals = k[c, t, h], v[c, t, h]
                if k_cur is not None:
                    tk, tv = k_cur[b, :, h].to(F64), v_cur[b, :, h].to(F64)
                    if cur_valid is not None:
                        m = cur_valid[b if cur_valid.shape[0] > 1 else 0].bool()[:tk.shape[0]]
                        tk, tv = tk[m], tv[m]
                    keys, vals = torch.cat([keys, tk]), torch.cat([vals, tv])
                if not len(keys):
                    continue
                i0, i1 = r * q_block, min((r + 1) * q_block, Lq)
                for x in range(G):
                    qq = q[b, i0:i1, h * G + x].to(F64)
                    s = qq @ keys.T * scale
                    e_s = 128 * 2.0 ** -24 * scale * (qq.abs() @ keys.T.abs()).amax(-1)
                    arg = 2.0 ** -23 * (s.amax(-1) - s.amin(-1) + s.abs().amax(-1)) * 1.45 + 2.0 ** -22
                    rel = e_s + arg
                    p = torch.softmax(s, -1)
                    hq = h * G + x
                    out[b, i0:i1, hq] = p @ vals
                    lse[b, hq, i0:i1] = torch.logsumexp(s, -1)
                    n = len(keys) * 2.0 ** -24
                    # fp16 probabilities and the sums of weight * value, then the bf16 output
                    tol_o[b, i0:i1, hq] = (2.0 ** -11 + 2 * rel[:, None] + 2 * n) * (p @ vals.abs()) + \
                        2.0 ** -8 * (1 + 2.0 ** -7) * (p @ vals).abs() + 2.0 ** -24
                    tol_l[b, hq, i0:i1] = rel + n + 2.0 ** -22 * (1 + lse[b, hq, i0:i1].abs())
    return out, lse, tol_o, tol_l


def _check_attention(got, ref, what):
    out, lse = got
    ro, rl, to, tl = ref
    assert torch.isfinite(out.float()).all(), what
    none = torch.isinf(rl)
    assert torch.equal(torch.isinf(lse), none) and (lse[none] < 0).all(), what
    assert (out.transpose(1, 2)[none] == 0).all(), what
    do, dl = (out.to(F64) - ro).abs() / to.clamp_min(2.0 ** -60), (lse.to(F64) - rl).abs()[~none] / tl[~none]
    print(f"[{what}] out {do.max().item() if do.numel() else 0:.3f} lse {dl.max().item() if dl.numel() else 0:.3f} of their bounds",
          flush=True)
    assert not do.numel() or do.max() <= 1, what
    assert not dl.numel() or dl.max() <= 1, what


def _lists(dev, B, H, runs, n, k, g, short=0):
    """Random ascending lists of k of n blocks; run r of every third head ends `short` entries early."""
    idx = torch.full((B, H, runs, k), -1, dtype=torch.int32, device=dev)
    m = min(k, n)
    if m:
        idx[..., :m] = torch.rand(B, H, runs, n, device=dev, generator=g).topk(m).indices.sort(-1).values.int()
    if short:
        idx[:, ::3, :, max(0, k - short):] = -1
    return idx


CASES = [
    # B, Lq, Hq, H, kv, block, q_block, K, Lc, fmt, holes, layout, slots
    (1, 1, 1, 1, 1, 64, 1, 1, 0, "fp8", 0, "bshd", 1),              # one query, one key
    (1, 1, 8, 2, 1000, 64, 1, 4, 1, "fp8", 0, "bshd", 1),           # single token, grouped heads
    (3, 1, 12, 2, 4097, 64, 1, 40, 0, "int8", 0.2, "bshd", 3),      # split keys, ragged end
    (2, 5, 24, 1, 700, 128, 2, 3, 9, "fp8", 0.5, "bshd", 2),        # 48 rows a run over one head
    (1, 33, 2, 2, 300, 64, 16, 3, 0, "fp8", 0, "bhsd", 1),
    (2, 200, 3, 3, 1500, 64, 64, 7, 130, "fp8", 0.1, "bshd", 1),    # one slot, ragged runs
    (1, 257, 4, 2, 2050, 256, 100, 5, 65, "int8", 0, "wide", 1),    # 200 rows a run: two tiles
    (1, 129, 2, 1, 640, 64, 128, 4, 129, "int8", 0.4, "bshd", 1),
    (1, 70, 2, 2, 0, 64, 64, 3, 70, "fp8", 0, "bshd", 1),           # no history yet
    (1, 64, 2, 2, 3000, 1024, 64, 2, 0, "fp8", 0.05, "bshd", 1),
    (1, 40, 3, 3, 500, 64, 8, 2, 3, "fp8", 0.97, "bshd", 1),        # masks that leave runs without a key
    (1, 3, 1, 1, 12800, 64, 1, 150, 0, "fp8", 0, "bshd", 1),        # lists of more than 64 entries: a row,
    (1, 20, 4, 2, 12800, 64, 16, 150, 33, "int8", 0.1, "bshd", 1),  # up to 64 rows,
    (1, 150, 1, 1, 12800, 64, 128, 150, 0, "fp8", 0.1, "bshd", 1),  # more
    (1, 100, 2, 2, 9000, 64, 50, 40, 70, "int8", 0.1, "bshd", 1),   # 50 rows a run: key halves by wave, split
    (1, 64, 1, 1, 200, 64, 64, 1, 65, "fp8", 0, "bshd", 1),         # one block, two tail tiles
    (1, 33, 2, 2, 130, 128, 64, 2, 64, "int8", 0, "wide", 1),
    (2, 11, 8, 2, 5000, 256, 11, 2, 1, "fp8", 0, "bhsd", 2),        # 44 rows of grouped heads
    (1, 64, 1, 1, 64, 64, 64, 1, 0, "fp8", 0, "bshd", 1),           # one tile in all
]


@pytest.mark.parametrize("B,Lq,Hq,H,kv,block,q_block,K,Lc,fmt,holes,layout,slots", CASES)
def test_attention_over_listed_blocks(dev, B, Lq, Hq, H, kv, block, q_block, K, Lc, fmt, holes, layout, slots):
    print(f"case sparse B={B} Lq={Lq} Hq={Hq}/{H} kv={kv} block={block} q_block={q_block} K={K} Lc={Lc} {fmt}",
          flush=True)
    ca = pkg_module("cache_attention")
    g = _gen(dev, Lq * 1000 + kv)
    cap = kv + 77
    cache = _cache(dev, slots, cap, H, fmt, g, layout)
    q = torch.randn(B, Lq, Hq, D, device=dev, generator=g).to(BF16)
    idx = _lists(dev, B, H, -(-Lq // q_block), -(-kv // block), K, g, short=1 if K > 2 else 0)
    valid = (torch.rand(slots, cap, device=dev, generator=g) >= holes) if holes else None
    k_cur = v_cur = cur_valid = None
    if Lc:
        k_cur = (torch.randn(B, Lc, H, D, device=dev, generator=g) * 1.5).to(BF16)
        v_cur = (torch.randn(B, Lc, H, D, device=dev, generator=g) * 1.5).to(BF16)
        if holes:
            cur_valid = torch.rand(B, Lc, device=dev, generator=g) >= holes
    ref = _attend(q, cache, kv, idx, block, q_block, k_cur, v_cur, valid, cur_valid)
    # what masked keys, unlisted rows past kv_len and masked tail keys hold does not matter
    unread = torch.zeros(slots, cap, dtype=torch.bool, device=dev)
    unread[:, kv:] = True
    if valid is not None:
        unread |= ~valid
    _poison(cache, unread)
    if cur_valid is not None:
        k_cur = torch.where(cur_valid[:, :, None, None], k_cur, INF)
        v_cur = torch.where(cur_valid[:, :, None, None], v_cur, float("nan"))
    got = ca.sparse_chunk_attention(q, cache, kv, idx, block=block, q_block=q_block, k_cur=k_cur, v_cur=v_cur,
                                    cache_valid=valid, cur_valid=cur_valid)
    _check_attention(got, ref, "listed blocks")


def test_attention_lists_at_their_edges(dev):
    """Empty lists, entries behind the first -1, past the last block and out of order,
    a block listed twice (its keys count twice), a list tensor with strides, K = 0."""
    ca = pkg_module("cache_attention")
    g = _gen(dev, 11)
    B, Lq, H, kv = 1, 96, 2, 500
    cache = _cache(dev, B, kv, H, "fp8", g)
    q = torch.randn(B, Lq, H, D, device=dev, generator=g).to(BF16)
    idx = torch.full((B, H, 3, 6), -1, dtype=torch.int32, device=dev)
    idx[0, 0, 0, :4] = torch.tensor([3, -1, 2, 1])
    idx[0, 0, 1] = torch.tensor([7, 6, 5, 0, 3, 2])
    idx[0, 0, 2, :3] = torch.tensor([0, 8, 2 ** 31 - 1])
    idx[0, 1, 0, :3] = torch.tensor([2, 2, 7])
    ref = _attend(q, cache, kv, idx.clamp_max(2 ** 20), 64, 32, None, None, None, None)
    got = ca.sparse_chunk_attention(q, cache, kv, idx, q_block=32)
    _check_attention(got, ref, "edges of lists")
    assert torch.isinf(got[1][0, 1, 32:]).all() and (got[0][0, 32:, 1] == 0).all()
    wide = torch.full((B, 3, H, 12), 5, dtype=torch.int32, device=dev)
    wide[:, :, :, :6] = idx.transpose(1, 2)
    again = ca.sparse_chunk_attention(q, cache, kv, wide[..., :6].transpose(1, 2), q_block=32)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    none = ca.sparse_chunk_attention(q, cache, kv, idx[..., :0], q_block=32)
    assert (none[0] == 0).all() and torch.isinf(none[1]).all()
    assert ca.sparse_chunk_attention(q[:, :0], cache, kv, idx[:, :, :0])[0].shape == (1, 0, H, D)


@pytest.mark.parametrize("Lq,kv,Lc,fmt", [(130, 1000, 0, "fp8"), (300, 513, 300, "int8"), (2, 9000, 2, "fp8"),
                                          (40, 0, 7, "fp8")])
def test_whole_cache_is_dense_attention(dev, Lq, kv, Lc, fmt):
    """Without a list, and with a list of every block: the dense attention's result."""
    ca = pkg_module("cache_attention")
    g = _gen(dev, kv + Lq)
    cache = _cache(dev, 1, max(kv, 1), 3, fmt, g)
    q = torch.randn(1, Lq, 3, D, device=dev, generator=g).to(BF16)
    k_cur = torch.randn(1, Lc, 3, D, device=dev, generator=g).to(BF16) if Lc else None
    v_cur = torch.randn(1, Lc, 3, D, device=dev, generator=g).to(BF16) if Lc else None
    ref = _attend(q, cache, kv, None, 64, 128, k_cur, v_cur, None, None)
    got = ca.sparse_chunk_attention(q, cache, kv, None, k_cur=k_cur, v_cur=v_cur)
    _check_attention(got, ref, "without a list")
    n, runs = -(-kv // 64), -(-Lq // 128)
    idx = torch.arange(n, dtype=torch.int32, device=dev).expand(1, 3, runs, n)
    _check_attention(ca.sparse_chunk_attention(q, cache, kv, idx, k_cur=k_cur, v_cur=v_cur), ref, "every block")
    dense = ca.chunk_attention(q, cache, kv, k_cur=k_cur, v_cur=v_cur)
    # both round their outputs to bf16 and their probabilities to fp16
    assert ((dense.to(F64) - ref[0]).abs() <= 2 * ref[2]).all()


@pytest.mark.parametrize("Lq", [1, 20, 50, 100])
def test_many_small_probabilities_beside_a_large_one(dev, Lq):
    """One key of every 32 (so one for each wave and split) takes nearly all the weight and
    holds V = 0; what the others, 2^-26 of it each, add up to is the whole output (_attend's
    bound is relative to it). A probability below the normal fp16 range is off by up to
    2^-25, where the largest ones, whose sum divides it, are 2^11 at least: 2^-36 a key
    over the number of large ones, on top."""
    ca = pkg_module("cache_attention")
    g = _gen(dev, 40 + Lq)
    H, n, gap = 2, 20000, 26 * math.log(2)
    e4m3 = torch.float8_e4m3fn
    cache = _cache(dev, 1, n, H, "fp8", g)
    unit = torch.zeros(D, device=dev)
    unit[0] = 1
    cache["k"].copy_((torch.randn(1, n, H, D, device=dev, generator=g) * 0.05).to(e4m3))
    cache["k"][:, ::32] = (unit * 16).to(e4m3)
    cache["v"].copy_((torch.rand(1, n, H, D, device=dev, generator=g) + 0.5).to(e4m3))
    cache["v"][:, ::32] = torch.zeros(D, device=dev).to(e4m3)
    cache["k_scale"].fill_(1.0)
    cache["v_scale"].fill_(64.0)
    # q . K is about 16 * 16 for those keys, near 0 for the others; the scale makes it the gap
    q = (unit * 16 + torch.randn(1, Lq, H, D, device=dev, generator=g) * 0.05).to(BF16)
    ref = _attend(q, cache, n, None, 64, Lq, None, None, None, None, scale=gap / 256)
    vals = _held(cache, "v")[0, :n].abs().sum(0)                       # [H, D]
    bound = ref[2] + 2.0 ** -36 * vals / (n // 32)
    blocks = torch.arange(-(-n // 64), dtype=torch.int32, device=dev).expand(1, H, 1, -1)
    for idx in (None, blocks):
        out, lse = ca.sparse_chunk_attention(q, cache, n, idx, q_block=Lq, softmax_scale=gap / 256)
        d = (out.to(F64) - ref[0]).abs() / bound
        print(f"[small probabilities {Lq}] {d.max().item():.3f} of the bound, output {ref[0].abs().mean():.2e}", flush=True)
        assert d.max() <= 1
        assert ((lse.to(F64) - ref[1]).abs() <= ref[3]).all()


def test_offsets_past_32_bits(dev):
    """A cache of more than 2^32 bytes a tensor, read, bounded, weighed and moved at its end."""
    ca, hist, kvc = pkg_module("cache_attention"), pkg_module("kv_history"), pkg_module("fp8_kv_cache")
    g = _gen(dev, 5)
    H, n = 24, 300
    cap = (1 << 32) // (H * D) + 40000                       # so many tokens that the codes pass 2^32 bytes
    big = kvc.make_fp8_kv_block(1, cap, H, D, device=dev)
    small = _cache(dev, 1, n, H, "fp8", g)
    start = (cap - n) // 64 * 64
    for name, t in small.items():
        big[name][:, start:start + n].copy_(t)
    kv = start + n
    assert start * H * D > 1 << 32
    q = torch.randn(1, 2, H, D, device=dev, generator=g).to(BF16)
    near = torch.arange(-(-n // 64), dtype=torch.int32, device=dev).expand(1, H, 1, -1)
    a = ca.sparse_chunk_attention(q, small, n, near, q_block=2)
    b = ca.sparse_chunk_attention(q, big, kv, near + start // 64, q_block=2)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    # the kernels of longer runs and of single rows, with and without holes
    near_valid = torch.rand(1, n, device=dev, generator=g) >= 0.3
    far_valid = torch.zeros(1, kv, dtype=torch.bool, device=dev)
    far_valid[:, start:] = near_valid
    for L in (1, 50, 100):
        ql = torch.randn(1, L, H, D, device=dev, generator=g).to(BF16)
        for nv, fv in ((None, None), (near_valid, far_valid)):
            c = ca.sparse_chunk_attention(ql, small, n, near, q_block=L, k_cur=ql, v_cur=ql, cache_valid=nv)
            d = ca.sparse_chunk_attention(ql, big, kv, near + start // 64, q_block=L, k_cur=ql, v_cur=ql, cache_valid=fv)
            assert all(torch.equal(x, y) for x, y in zip(c, d)), L
    bounds = hist.make_block_bounds(big)
    hist.update_block_bounds(bounds, big, start, kv)
    ref = hist.make_block_bounds(small)
    hist.update_block_bounds(ref, small, 0, n)
    assert torch.equal(bounds[:, start // 64:start // 64 + ref.shape[1]], ref)
    assert torch.isinf(bounds[:, :start // 64].float()).all()
    valid = torch.zeros(1, kv, dtype=torch.bool, device=dev)
    valid[:, start:] = True
    mass = hist.key_mass(q, a[1], big, kv, cache_valid=valid)
    assert (mass[:, :, :start] == 0).all()
    assert torch.equal(mass[:, :, start:], hist.key_mass(q, a[1], small, n))
    out = kvc.make_fp8_kv_block(1, n, H, D, device=dev)
    idx, _ = hist.evict(big, out, mass, kv, n, cache_valid=valid)
    assert torch.equal(idx, torch.arange(start, kv, dtype=torch.int32, device=dev).expand(1, H, n))
    for name, t in small.items():
        assert torch.equal(out[name].view(torch.uint8), t.view(torch.uint8))


# --------------------------------------------------------------------------
# key mass

@pytest.mark.parametrize("Bq,slots,Lq,Hq,H,kv,fmt,holes,layout,prior", [
    (1, 1, 1, 1, 1, 1, "fp8", 0, "bshd", 0),
    (2, 2, 1, 8, 2, 1000, "fp8", 0.3, "bshd", 700),       # single tokens of grouped heads
    (3, 1, 40, 2, 2, 300, "int8", 0, "bshd", 300),        # one slot draws from three batches
    (1, 1, 33, 3, 3, 257, "fp8", 0.1, "bhsd", 0),
    (1, 1, 2000, 2, 1, 70, "int8", 0.2, "wide", 64),      # few keys, many rows: split rows
    (2, 2, 700, 3, 3, 513, "fp8", 0, "bshd", 1),
    (1, 1, 3, 16, 8, 70001, "fp8", 0.1, "bshd", 69000),     # few rows, several steps of keys a workgroup
    (4, 1, 4, 4, 2, 33333, "int8", 0, "bhsd", 0),           # 32 rows of four batches over one slot
    (1, 1, 0, 2, 2, 100, "fp8", 0, "bshd", 60),           # no query: the prior alone
])
def test_key_mass(dev, Bq, slots, Lq, Hq, H, kv, fmt, holes, layout, prior):
    print(f"case mass B={Bq}/{slots} Lq={Lq} Hq={Hq}/{H} kv={kv} {fmt} {layout}", flush=True)
    hist, ca = pkg_module("kv_history"), pkg_module("cache_attention")
    g = _gen(dev, Lq + kv)
    cache = _cache(dev, slots, kv + 50, H, fmt, g, layout)
    q = torch.randn(Bq, Lq, Hq, D, device=dev, generator=g).to(BF16)
    valid = (torch.rand(slots, kv + 3, device=dev, generator=g) >= holes) if holes else None
    before = torch.rand(slots, H, prior + 5, device=dev, generator=g)[:, :, :prior] if prior else None
    _, lse = ca.sparse_chunk_attention(q, cache, kv, None, cache_valid=valid)
    if Lq > 5:                                             # rows that add nothing, whatever they hold
        lse[:, :, 3], lse[:, :, 5] = -INF, INF
        q[:, 3] = float("nan")
        q[:, 5] = INF
    G, k = Hq // H, _held(cache, "k")[:, :kv]
    ref = torch.zeros(slots, H, kv, dtype=F64, device=dev)
    tol = torch.zeros_like(ref)
    for b in range(Bq):
        c = b if slots == Bq else 0
        for hq in range(Hq):
            rows = torch.isfinite(lse[b, hq])
            qq, ll = q[b, rows, hq].to(F64), lse[b, hq, rows].to(F64)[:, None]
            s = qq @ k[c, :, hq // G].T * SCALE
            p = torch.exp(s - ll)
            e = 128 * 2.0 ** -24 * SCALE * (qq.abs() @ k[c, :, hq // G].T.abs()) + 2.0 ** -23 * 1.45 * (s.abs() + 2 * ll.abs()) \
                + 2.0 ** -22
            ref[c, hq // G] += p.sum(0)
            tol[c, hq // G] += (p * e).sum(0)
    tol += ref * (Bq * Lq * G) * 2.0 ** -24
    if valid is not None:
        ref *= valid[:, None, :kv]
    if prior:
        ref[:, :, :prior] += before.to(F64)
    tol += ref * 2.0 ** -23 + 2.0 ** -126
    unread = torch.zeros(slots, kv + 50, dtype=torch.bool, device=dev)
    unread[:, kv:] = True
    if valid is not None:
        unread[:, :kv] |= ~valid[:, :kv]
    _poison(cache, unread)
    got = hist.key_mass(q, lse, cache, kv, prior=before, cache_valid=valid)
    worst = ((got.to(F64) - ref).abs() / tol).max().item()
    print(f"[mass] {worst:.3f} of its bound", flush=True)
    assert worst <= 1
    assert torch.equal(got, hist.key_mass(q, lse, cache, kv, prior=before, cache_valid=valid))   # no order to vary


def test_key_mass_counts_every_row(dev):
    """Dense rows of finite log-sum-exp each give 1 in all to the keys they read."""
    hist, ca = pkg_module("kv_history"), pkg_module("cache_attention")
    g = _gen(dev, 9)
    cache = _cache(dev, 1, 1500, 4, "fp8", g)
    q = torch.randn(1, 333, 8, D, device=dev, generator=g).to(BF16)
    _, lse = ca.sparse_chunk_attention(q, cache, 1500, None)
    total = hist.key_mass(q, lse, cache, 1500).to(F64).sum(-1)
    # each of the 666 rows' weights is off by the logits' and the exponent's roundings (2^-16 for these sizes)
    assert ((total - 666).abs() <= 666 * 2.0 ** -16).all()


# --------------------------------------------------------------------------
# eviction

def _evict_reference(mass, kv, keep, first, last, valid):
    B, H = mass.shape[:2]
    m = mass.cpu().double()
    out = []
    for b in range(B):
        for h in range(H):
            s = [x if x == x else -INF for x in m[b, h, :kv].tolist()]
            empty = [valid is not None and not bool(valid[b if valid.shape[0] > 1 else 0, t]) for t in range(kv)]
            out.append(_choose(s, [t < first or t >= kv - last for t in range(kv)], empty, keep))
    return torch.tensor(out, dtype=torch.int32).reshape(B, H, keep)


def test_select_tokens_equal_masses(dev):
    """Rows of one value, and of two: the lowest indices, in short and long rows."""
    hist = pkg_module("kv_history")
    for n in (10, 9000, 33001):
        mass = torch.zeros(1, 2, n, device=dev)
        mass[0, 1, n // 2:] = 1e-30
        got = hist.select_tokens(mass, n, n // 2 + 3, keep_last=1).cpu()
        want = [*range(n // 2 + 2), n - 1]
        assert got[0, 0].tolist() == want
        high = list(range(n // 2, n))
        want = sorted(high + list(range(n // 2 + 3 - len(high))))[:n // 2 + 3]
        assert got[0, 1].tolist() == want, n


@pytest.mark.parametrize("B,H,kv,keep,first,last,fmt,holes,layout", [
    (1, 1, 1, 1, 0, 0, "fp8", 0, "bshd"),
    (2, 3, 1000, 400, 16, 100, "fp8", 0, "bshd"),
    (1, 24, 2049, 1024, 0, 0, "int8", 0.1, "bshd"),
    (2, 2, 300, 250, 10, 10, "int8", 0.6, "bhsd"),        # fewer valid tokens than places
    (1, 5, 129, 200, 0, 3, "fp8", 0, "wide"),             # more places than tokens
    (1, 2, 5000, 7, 7, 0, "fp8", 0, "bshd"),              # only the first
    (1, 2, 64, 0, 0, 0, "fp8", 0, "bshd"),
    (1, 3, 0, 5, 0, 0, "fp8", 0, "bshd"),
    (1, 2, 32769, 20000, 5, 300, "fp8", 0.02, "bshd"),    # past one workgroup a head
    (2, 1, 70001, 123, 0, 1, "int8", 0, "bshd"),
    (1, 1, 40000, 39000, 0, 0, "fp8", 0.5, "bshd"),       # long, and fewer valid tokens than places
    (1, 1, 33000, 40000, 10, 10, "fp8", 0, "bshd"),       # long, and more places than tokens
    (1, 2, 20000, 9000, 0, 64, "fp8", 0, "bshd"),
])
def test_evict(dev, B, H, kv, keep, first, last, fmt, holes, layout):
    print(f"case evict B={B} H={H} kv={kv} keep={keep} {first}/{last} {fmt} {layout}", flush=True)
    hist, kvc = pkg_module("kv_history"), pkg_module("fp8_kv_cache")
    g = _gen(dev, kv + keep)
    cache = _cache(dev, B, kv + 11, H, fmt, g, layout)
    # a mass in few values, so that ties decide, with zeros of both signs, NaN and infinities
    mass = torch.randint(0, max(2, kv // 8), (B, H, kv + 5), device=dev, generator=g).float() / 7
    special = torch.tensor([0.0, -0.0, float("nan"), INF, -INF, 1e-42], device=dev)
    at = torch.randint(0, 40, mass.shape, device=dev, generator=g)
    mass = torch.where(at < 6, special[at.clamp_max(5)], mass)
    valid = (torch.rand(B, kv, device=dev, generator=g) >= holes) if holes else None
    make = kvc.make_fp8_kv_block if fmt == "fp8" else kvc.make_int8_kv_block
    out = make(B, keep + 6, H, D, device=dev)
    for t in out.values():
        t.view(torch.uint8).fill_(0x5a)
    idx, moved = hist.evict(cache, out, mass, kv, keep, keep_first=first, keep_last=last, cache_valid=valid)
    ref = _evict_reference(mass, kv, keep, first, last, valid)
    assert torch.equal(idx.cpu(), ref)
    there = (idx >= 0)
    assert torch.equal(there[:, :1].expand_as(there), there)     # as many in every head
    bi, hi = torch.arange(B, device=dev)[:, None, None], torch.arange(H, device=dev)[None, :, None]
    for name, t in out.items():
        src = cache[name].view(torch.uint8)
        want = torch.full_like(t.view(torch.uint8), 0x5a)
        if kv and keep:
            rows = torch.where(there[..., None], src[bi, idx.long().clamp_min(0), hi], 0x5a)
            want[:, :keep] = rows.transpose(1, 2)
        assert torch.equal(t.view(torch.uint8), want), name       # rows behind the last: as they were
    if kv and keep:
        want = torch.where(there, mass[bi, hi, idx.long().clamp_min(0)], 0.0)
        assert torch.equal(moved.view(torch.int32), want.view(torch.int32))


def test_evict_refuses_its_own_cache(dev):
    hist = pkg_module("kv_history")
    cache = _cache(dev, 1, 100, 2, "fp8", _gen(dev, 1))
    mass = torch.rand(1, 2, 100, device=dev)
    with pytest.raises(RuntimeError, match="overlaps"):
        hist.evict(cache, cache, mass, 100, 50)
    with pytest.raises(RuntimeError, match="overlaps"):
        hist.evict({n: t[:, :60] for n, t in cache.items()}, {n: t[:, 40:] for n, t in cache.items()}, mass[..., :60], 60, 30)


def test_evict_of_an_empty_cache(dev):
    """No token, no mass: every place stays empty and the output as it was."""
    hist, kvc = pkg_module("kv_history"), pkg_module("fp8_kv_cache")
    for cap in (0, 20):
        cache, out = kvc.make_fp8_kv_block(2, cap, 3, D, device=dev), kvc.make_fp8_kv_block(2, 8, 3, D, device=dev)
        for t in out.values():
            t.view(torch.uint8).fill_(0x5a)
        idx, moved = hist.evict(cache, out, torch.empty(2, 3, 0, device=dev), 0, 6)
        assert idx.shape == (2, 3, 6) and (idx == -1).all() and moved.shape == (2, 3, 6) and (moved == 0).all()
        assert all((t.view(torch.uint8) == 0x5a).all() for t in out.values())


# --------------------------------------------------------------------------
# together

def _round(dev, q, k, v, cache, out, bounds, state):
    """A chunk as a program runs it: sparse pass, dense write pass with mass, write, cut."""
    hist, ca, kvc = pkg_module("kv_history"), pkg_module("cache_attention"), pkg_module("fp8_kv_cache")
    kv, L = state["kv"], q.shape[1]
    idx = hist.select_blocks(q, bounds, kv, 6, q_block=64, keep_first=1, keep_last=2)
    near, _ = ca.sparse_chunk_attention(q, cache, kv, idx, q_block=64, k_cur=k, v_cur=v)
    full, lse = ca.sparse_chunk_attention(q, cache, kv, None, k_cur=k, v_cur=v)
    kvc.quantize_kv_pair_into(cache, k, v, kv, status=state["status"])
    hist.update_block_bounds(bounds, cache, kv, kv + L)
    mass = hist.key_mass(q, lse, cache, kv + L, prior=state["mass"])
    kept, moved = hist.evict(cache, out, mass, kv + L, 900, keep_first=64, keep_last=L)
    fresh = hist.make_block_bounds(out)
    hist.update_block_bounds(fresh, out, 0, 900)
    again = hist.select_blocks(q, fresh, 900, 6, q_block=64, keep_first=1, keep_last=2)
    last, _ = ca.sparse_chunk_attention(q, out, 900, again, q_block=64)
    return idx, near, full, lse, mass, kept, moved, fresh, again, last


def test_a_chunk_with_its_operators_together(dev):
    """The run in one: eager against 64 bits at its ends, on another stream, and in a
    graph replayed on new inputs with eager work between the replays."""
    hist, kvc = pkg_module("kv_history"), pkg_module("fp8_kv_cache")
    g = _gen(dev, 21)
    H, kv, L = 4, 1000, 200
    cache = _cache(dev, 1, kv + L, H, "fp8", g)
    out = kvc.make_fp8_kv_block(1, 1000, H, D, device=dev)
    bounds = hist.make_block_bounds(cache)
    hist.update_block_bounds(bounds, cache, 0, kv)
    state = dict(kv=kv, mass=torch.rand(1, H, kv, device=dev, generator=g),
                 status=torch.zeros(1, dtype=torch.int32, device=dev))

    def inputs(seed):
        gg = _gen(dev, seed)
        return [torch.randn(1, L, H, D, device=dev, generator=gg).to(BF16) for _ in range(3)]

    q, k, v = inputs(1)
    ref = _attend(q, cache, kv, None, 64, 64, k, v, None, None)
    with torch.no_grad():
        eager = _round(dev, q, k, v, cache, out, bounds, state)
        _check_attention((eager[2], eager[3]), ref, "dense pass")
        assert torch.equal(eager[0].cpu(), _select_reference(q, bounds, kv, 6, 64, 64, 1, 2, None))
        ref = _attend(q, cache, kv, eager[0], 64, 64, k, v, None, None)
        assert ((eager[1].to(F64) - ref[0]).abs() <= ref[2]).all()
        assert torch.equal(eager[5].cpu(), _evict_reference(eager[4], kv + L, 900, 64, L, None))
        ref = _attend(q, out, 900, eager[8], 64, 64, None, None, None, None)
        assert ((eager[9].to(F64) - ref[0]).abs() <= ref[2]).all()

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = _round(dev, q, k, v, cache, out, bounds, state)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, other))

        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = _round(dev, q, k, v, cache, out, bounds, state)
        for seed in (2, 3, 4, 5):
            for dst, src in zip((q, k, v), inputs(seed)):
                dst.copy_(src)
            graph.replay()
            torch.cuda.synchronize()
            replayed = [t.clone() for t in held]
            eager = _round(dev, q, k, v, cache, out, bounds, state)
            for i, (a, b) in enumerate(zip(replayed, eager)):
                assert torch.equal(a, b), (seed, i)
    assert int(state["status"]) == 0


def test_compiled_callers_hold_the_ops(dev):
    """torch.compile keeps each op as one node; a dispatch mode sees them."""
    hist, ca = pkg_module("kv_history"), pkg_module("cache_attention")
    g = _gen(dev, 31)
    cache = _cache(dev, 1, 640, 2, "fp8", g)
    q = torch.randn(1, 100, 2, D, device=dev, generator=g).to(BF16)

    def step(q, bounds):
        hist.update_block_bounds(bounds, cache, 0, 640)
        idx = hist.select_blocks(q, bounds, 640, 3, q_block=50)
        out, lse = ca.sparse_chunk_attention(q, cache, 640, idx, q_block=50)
        return out, hist.key_mass(q, lse, cache, 640)

    with torch.no_grad():
        eager = step(q, hist.make_block_bounds(cache))
        torch._dynamo.reset()
        compiled = torch.compile(step, backend="aot_eager", fullgraph=True)(q, hist.make_block_bounds(cache))
    assert all(torch.equal(a, b) for a, b in zip(eager, compiled))


def test_layer_history_of_one_slot(dev):
    """One history slot read by three query batches of grouped heads: lists of each batch,
    the weight of all of them on one mass, an eviction, and a pass over what it left."""
    hist, kvc = pkg_module("kv_history"), pkg_module("fp8_kv_cache")
    g = _gen(dev, 61)
    B, H, kv, L = 3, 2, 600, 70
    cache = _cache(dev, 1, 800, H, "int8", g)
    out = kvc.make_int8_kv_block(1, 800, H, D, device=dev)
    h = hist.LayerHistory(cache, top_k=4, q_block=32, keep_first=1, keep_last=1, track_mass=True)
    h.reset(cache, kv)
    q = torch.randn(B, L, 2 * H, D, device=dev, generator=g).to(BF16)
    k, v = (torch.randn(B, L, H, D, device=dev, generator=g).to(BF16) for _ in range(2))
    idx = hist.select_blocks(q, h.bounds, kv, 4, q_block=32, keep_first=1, keep_last=1)
    assert torch.equal(idx.cpu(), _select_reference(q, h.bounds, kv, 4, 64, 32, 1, 1, None))
    ref = _attend(q, cache, kv, idx, 64, 32, k, v, None, None)
    assert ((h.attend(q, k, v, cache, kv, False).to(F64) - ref[0]).abs() <= ref[2]).all()
    assert h.length == kv and (h.mass == 0).all()
    # a writing pass: its tokens are in the cache already; its queries' weight counts once committed
    ref = _attend(q, cache, kv, None, 64, L, k, v, None, None)
    assert ((h.attend(q, k, v, cache, kv, True).to(F64) - ref[0]).abs() <= ref[2]).all()
    assert h.length == kv
    h.commit(cache)
    keys = _held(cache, "k")[0, :kv + L]
    want = torch.zeros(H, kv + L, dtype=F64, device=dev)
    for b in range(B):
        for hq in range(2 * H):
            s = q[b, :, hq].to(F64) @ keys[:, hq // 2].T * SCALE
            want[hq // 2] += (s - ref[1][b, hq][:, None]).exp().sum(0)
    # an exponent is off by its logit's fp32 sum, the log-sum-exp's bound and the argument's
    # rounding; each of the rows' terms adds half a step to its sum
    worst = (q.to(F64).abs().amax() * keys.abs().sum(-1).amax() * SCALE).item()
    rel = 128 * 2.0 ** -24 * worst + ref[3].max().item() + 2.0 ** -22 * (1 + worst)
    assert h.length == kv + L and h.mass.shape == (1, H, kv + L)
    assert ((h.mass[0].to(F64) - want).abs() <= (rel + 2 * B * L * 2 * 2.0 ** -24) * want).all()
    kept = h.evict(cache, out, kv + L, 400, keep_first=10, keep_last=L)
    assert kept.shape == (1, H, 400) and h.length == 400 and h.mass.shape == (1, H, 400)
    ref = _attend(q, out, 400, hist.select_blocks(q, h.bounds, 400, 4, q_block=32, keep_first=1, keep_last=1), 64, 32,
                  k, v, None, None)
    assert ((h.attend(q, k, v, out, 400, False).to(F64) - ref[0]).abs() <= ref[2]).all()


# --------------------------------------------------------------------------
# the AR model's long roll-outs

def _model(dev, **kw):
    dit = pkg_module("dit_block")
    return dit.FP8ARModel(depth=2, hidden=256, heads=2, latent_shape=(1, 8, 16), max_chunks=4, device=dev, seed=3, **kw)


def _chunk(dev, seed):
    g = _gen(dev, seed)
    noise = torch.randn(1, 128, 256, device=dev, generator=g).to(BF16)
    vecs = [torch.randn(1, 256, device=dev, generator=g).to(BF16) for _ in range(3)]
    return noise, vecs[:2], vecs[2], [1.0, 0.5, 0.0]


def test_model_with_enough_blocks_is_the_dense_model(dev):
    """A history of no more blocks than top_k is read whole: the same outputs, bit for bit."""
    dense, sparse = _model(dev), _model(dev, sparse_top_k=8)
    for i in range(4):
        a, b = dense.generate_chunk(*_chunk(dev, i)), sparse.generate_chunk(*_chunk(dev, i))
        assert torch.equal(a, b), i


def test_model_reads_blocks_and_cuts_a_full_cache(dev):
    """Denoising passes read the chosen blocks; a full cache is cut to the heaviest
    tokens and the roll-out goes on; a refused write leaves bounds and mass alone."""
    hist = pkg_module("kv_history")
    m = _model(dev, sparse_top_k=3, evict_keep=300)
    plain = _model(dev)
    for i in range(4):
        out = m.generate_chunk(*_chunk(dev, i))
        assert torch.isfinite(out.float()).all() and m.cache_valid_len == 128 * (i + 1)
        plain.generate_chunk(*_chunk(dev, i))
    with pytest.raises(ValueError, match="capacity"):
        plain.generate_chunk(*_chunk(dev, 9))
    for h, c in zip(m.histories, m.caches):
        assert h.mass.shape == (1, 2, 512) and torch.isfinite(h.mass).all() and (h.mass > 0).all()
        ref = hist.make_block_bounds(c)
        hist.update_block_bounds(ref, c, 0, 512)
        assert torch.equal(h.bounds, ref)
    # a layer's attention over chosen blocks, against the plain form
    g = _gen(dev, 77)
    q, k, v = (torch.randn(1, 128, 2, D, device=dev, generator=g).to(BF16) for _ in range(3))
    h, c = m.histories[0], m.caches[0]
    idx = hist.select_blocks(q, h.bounds, 512, 3, keep_first=1, keep_last=2)
    assert (idx == torch.tensor([0, 6, 7], device=dev)).all()   # three places, all spoken for
    ref = _attend(q, c, 512, idx, 64, 128, k, v, None, None)
    assert ((h.attend(q, k, v, c, 512, False).to(F64) - ref[0]).abs() <= ref[2]).all()
    # the fifth chunk cuts the history first
    before = [{n: t.clone() for n, t in c.items()} for c in m.caches]
    mass = [h.mass.clone() for h in m.histories]
    noise, vecs, vec, sigmas = _chunk(dev, 4)
    out = m.generate_chunk(noise, vecs, vec, sigmas)
    assert torch.isfinite(out.float()).all() and m.cache_valid_len == 300 + 128
    for i, c in enumerate(m.caches):
        kept = _evict_reference(mass[i], 512, 300, 75, 128, None).to(dev).long()
        for name, t in c.items():
            want = before[i][name].transpose(1, 2).gather(2, kept[..., None].expand(-1, -1, -1, t.shape[3])) \
                if t.dtype == torch.float32 else \
                before[i][name].view(torch.uint8).transpose(1, 2).gather(2, kept[..., None].expand(-1, -1, -1, t.shape[3]))
            got = t[:, :300].transpose(1, 2)
            assert torch.equal(got if t.dtype == torch.float32 else got.view(torch.uint8), want), name
    # a write that is refused: after it (and the cut that made room for it) nothing moves
    with torch.no_grad():
        m.blocks[1].qkv.bias[300] = float("nan")
    with pytest.raises(ValueError, match="non-finite"):
        m.generate_chunk(noise, [], vec, [1.0])
    assert m.cache_valid_len == 300
    bounds, mass = [h.bounds.clone() for h in m.histories], [h.mass.clone() for h in m.histories]
    with pytest.raises(ValueError, match="non-finite"):
        m.generate_chunk(noise, [], vec, [1.0])
    assert m.cache_valid_len == 300
    for h, b, w in zip(m.histories, bounds, mass):
        assert torch.equal(h.bounds, b) and torch.equal(h.mass, w) and h.mass.shape == (1, 2, 300)


def test_model_starts_a_new_roll_out(dev):
    """A second roll-out over the same caches is the first one again: nothing of the old
    history's mass or bounds is left; filled caches are taken in by reset."""
    hist = pkg_module("kv_history")
    m = _model(dev, sparse_top_k=3, evict_keep=300)
    first = [m.generate_chunk(*_chunk(dev, i)) for i in range(5)]
    mass = [h.mass for h in m.histories]
    m.cache_valid_len = m.frames_done = 0
    again = [m.generate_chunk(*_chunk(dev, i)) for i in range(5)]
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    assert all(torch.equal(a, h.mass) for a, h in zip(mass, m.histories))
    h, c = m.histories[0], m.caches[0]
    m.cache_valid_len = 100                               # moved by hand: refused until taken in
    with pytest.raises(ValueError, match="accounts for 428 tokens, the pass reads 100"):
        m.generate_chunk(*_chunk(dev, 5))
    for h, c in zip(m.histories, m.caches):
        h.reset(c, 100)
        ref = hist.make_block_bounds(c)
        hist.update_block_bounds(ref, c, 0, 100)
        assert torch.equal(h.bounds[:, :2], ref[:, :2]) and (h.mass == 0).all() and h.mass.shape == (1, 2, 100)
    assert torch.isfinite(m.generate_chunk(*_chunk(dev, 5)).float()).all()


def test_model_refusals(dev):
    for kw in (dict(sparse_top_k=-1), dict(evict_keep=-1), dict(evict_keep=385), dict(sparse_top_k=1, text_len=8)):
        with pytest.raises(ValueError):
            _model(dev, **kw)
    with pytest.raises(ValueError, match="evict_keep"):
        _model(dev).evict_history()


# --------------------------------------------------------------------------
# every kernel of the dispatch, at the sizes that reach it

@pytest.mark.parametrize("B,Lq,Hq,H,kv,block,q_block,K,Lc,fmt,holes,layout,slots", [
    (1, 1, 3, 3, 700, 64, 1, 5, 40, "int8", 0.3, "bshd", 1),        # one row a run: holes in cache and tail
    (2, 3, 2, 2, 4097, 128, 1, 20, 70, "fp8", 0.2, "wide", 2),      # split, a ragged last block, two tail tiles
    (2, 2, 5, 5, 20000, 64, 1, 300, 0, "int8", 0, "bhsd", 1),       # split over many tiles, one slot
    (1, 9, 2, 2, 300, 64, 1, 3, 1, "int8", 0.95, "bshd", 1),        # hardly a key left
    (1, 4, 1, 1, 0, 64, 1, 2, 131, "fp8", 0.4, "bshd", 1),          # the tail alone
])
def test_attention_of_single_rows(dev, B, Lq, Hq, H, kv, block, q_block, K, Lc, fmt, holes, layout, slots):
    test_attention_over_listed_blocks(dev, B, Lq, Hq, H, kv, block, q_block, K, Lc, fmt, holes, layout, slots)


@pytest.mark.parametrize("Lq,q_block", [(3, 1), (20, 20), (50, 50), (100, 100)])
def test_attention_over_a_tail_past_31_bits(dev, Lq, q_block):
    """Tail tokens so far apart that the rows of a head span more than 2^31 bytes: every
    kernel (by rows a run) gives what it gives for the same tail laid out densely."""
    ca = pkg_module("cache_attention")
    g = _gen(dev, 60 + Lq)
    H, kv, Lc, far = 2, 300, 71, 0xfffff8
    assert (Lc * far + D) * 2 >= 1 << 31
    cache = _cache(dev, 1, kv, H, "fp8", g)
    q = torch.randn(1, Lq, H, D, device=dev, generator=g).to(BF16)
    buf = torch.full(((Lc - 1) * far + 2 * H * D,), float("nan"), dtype=BF16, device=dev)
    k_far, v_far = (buf.as_strided((1, Lc, H, D), (Lc * far, far, D, 1), i * H * D) for i in (0, 1))
    k_far.copy_(torch.randn(1, Lc, H, D, device=dev, generator=g).to(BF16))
    v_far.copy_(torch.randn(1, Lc, H, D, device=dev, generator=g).to(BF16))
    k, v = k_far.contiguous(), v_far.contiguous()
    idx = torch.tensor([4, 0, 1], dtype=torch.int32, device=dev).expand(1, H, -(-Lq // q_block), 3)
    for u in (None, torch.rand(1, Lc, device=dev, generator=g) >= 0.3):
        print(f"case far tail Lq={Lq} masked={u is not None}", flush=True)
        kw = dict(q_block=q_block, cur_valid=u)
        near = ca.sparse_chunk_attention(q, cache, kv, idx, k_cur=k, v_cur=v, **kw)
        _check_attention(near, _attend(q, cache, kv, idx, 64, q_block, k, v, None, u), "dense tail")
        far_ = ca.sparse_chunk_attention(q, cache, kv, idx, k_cur=k_far, v_cur=v_far, **kw)
        assert all(torch.equal(a, b) for a, b in zip(near, far_))


@pytest.mark.parametrize("Lq,q_block", [(3, 1), (20, 20), (50, 50), (100, 100)])
def test_attention_repeats_itself(dev, Lq, q_block):
    """Splits are merged in their order: the same call gives the same bits."""
    ca = pkg_module("cache_attention")
    g = _gen(dev, 80 + Lq)
    cache = _cache(dev, 1, 9000, 3, "int8", g)
    q = torch.randn(1, Lq, 3, D, device=dev, generator=g).to(BF16)
    valid = torch.rand(1, 9000, device=dev, generator=g) >= 0.1
    idx = _lists(dev, 1, 3, -(-Lq // q_block), 141, 60, g)
    first = ca.sparse_chunk_attention(q, cache, 9000, idx, q_block=q_block, k_cur=q, v_cur=q, cache_valid=valid)
    for _ in range(5):
        again = ca.sparse_chunk_attention(q, cache, 9000, idx, q_block=q_block, k_cur=q, v_cur=q, cache_valid=valid)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("Lq,Hq,H,n,q_block,top_k,first,last,gone", [
    (1, 2, 1, 2048, 1, 64, 1, 2, 0.1),        # the last size with 8 elements a thread,
    (1, 2, 1, 2049, 1, 64, 1, 2, 0.1),        # the first and the last with 32,
    (2, 2, 2, 8192, 1, 300, 0, 1, 0),
    (2, 1, 1, 8193, 1, 300, 3, 0, 0.3),       # rows read again in every pass
    (1, 1, 1, 10001, 1, 9000, 1, 1, 0.2),     # (more places than blocks)
    (1, 1, 1, 10001, 1, 1, 0, 0, 0),
    (544, 2, 2, 600, 32, 30, 2, 2, 0.1),      # 17 runs: two run tiles, three stretches of blocks
    (40, 2, 1, 2049, 8, 100, 1, 1, 0),        # many runs in the longer searches
    (20, 1, 1, 8193, 4, 77, 0, 2, 0.05),
])
@pytest.mark.parametrize("ties", [False, True])
def test_select_of_many_blocks(dev, Lq, Hq, H, n, q_block, top_k, first, last, gone, ties):
    """ties: small whole numbers, of which many blocks have the score of the last place."""
    print(f"case select Lq={Lq} Hq={Hq}/{H} blocks={n} q_block={q_block} k={top_k} ties={ties}", flush=True)
    hist = pkg_module("kv_history")
    g = _gen(dev, Lq + n + top_k)
    if ties:
        q = torch.randint(-1, 2, (1, Lq, Hq, D), device=dev, generator=g).to(BF16)
        lo = torch.randint(-1, 1, (1, n, H, 1, D), device=dev, generator=g)
        bounds = torch.cat([lo, lo + torch.randint(0, 2, (1, n, H, 1, D), device=dev, generator=g)], 3).to(BF16)
    else:
        q = torch.randn(1, Lq, Hq, D, device=dev, generator=g).to(BF16)
        bounds = _random_bounds(dev, 1, n, H, g)
    if gone:
        no = torch.rand(1, n, device=dev, generator=g) < gone
        bounds[:, :, :, 0] = torch.where(no[:, :, None, None], INF, bounds[:, :, :, 0])
        bounds[:, :, :, 1] = torch.where(no[:, :, None, None], -INF, bounds[:, :, :, 1])
    got = hist.select_blocks(q, bounds, n * 64 - 9, top_k, q_block=q_block, keep_first=first, keep_last=last)
    # whole numbers: exact; else a 64-bit sum is off by 2^-44 of its magnitudes at most, which
    # changes a choice only between two scores at the last place that are as close
    assert torch.equal(got.cpu(), _select_reference(q, bounds, n * 64 - 9, top_k, 64, q_block, first, last, None))


@pytest.mark.parametrize("Bq,slots,Lq,Hq,H,kv,fmt,holes,layout,prior", [
    (1, 1, 33, 24, 24, 11009, "fp8", 0.1, "bshd", 11009),   # 512 keys a workgroup, a ragged last one
    (3, 1, 40, 24, 24, 11000, "int8", 0, "bshd", 9001),     # three batches over one slot
    (2, 2, 17, 48, 24, 5600, "int8", 0.3, "wide", 0),       # grouped heads, rows of two heads
    (1, 1, 65, 8, 8, 40000, "fp8", 0.97, "bhsd", 700),
])
def test_key_mass_of_long_caches(dev, Bq, slots, Lq, Hq, H, kv, fmt, holes, layout, prior):
    assert slots * H * -(-kv // 512) >= 2 * torch.cuda.get_device_properties(dev).multi_processor_count
    test_key_mass(dev, Bq, slots, Lq, Hq, H, kv, fmt, holes, layout, prior)


def test_model_cuts_every_layer_or_none(dev):
    """A layer that cannot be cut (its mass is of other tokens, or missing) leaves the
    layers before it as they were; put right, the roll-out goes on."""
    m = _model(dev, sparse_top_k=3, evict_keep=300)
    for i in range(4):
        m.generate_chunk(*_chunk(dev, i))
    caches, spare = list(m.caches), m.spare
    held = [{n: t.clone() for n, t in c.items()} for c in caches]
    mass, bounds = [h.mass.clone() for h in m.histories], [h.bounds.clone() for h in m.histories]
    last = m.histories[-1]
    whole = (last.length, last.mass)
    for spoiled, message in (((500, last.mass), "accounts for 500 tokens, not 512"), ((512, None), "needs the mass")):
        last.length, last.mass = spoiled
        for call in (m.evict_history, lambda: m.generate_chunk(*_chunk(dev, 4))):
            with pytest.raises(ValueError, match=message):
                call()
        last.length, last.mass = whole
        assert m.cache_valid_len == 512 and m.spare is spare and all(a is b for a, b in zip(m.caches, caches))
        for c, old in zip(m.caches, held):
            assert all(torch.equal(c[n].view(torch.uint8), old[n].view(torch.uint8)) for n in old)
        for h, w, b in zip(m.histories, mass, bounds):
            assert h.length == 512 and torch.equal(h.mass, w) and torch.equal(h.bounds, b)
    assert torch.isfinite(m.generate_chunk(*_chunk(dev, 4)).float()).all() and m.cache_valid_len == 300 + 128


def test_model_keeps_the_history_of_a_refused_call(dev):
    """Arguments are looked at before a full cache is cut."""
    m = _model(dev, evict_keep=300)
    for i in range(4):
        m.generate_chunk(*_chunk(dev, i))
    caches, mass = list(m.caches), [h.mass.clone() for h in m.histories]
    noise, vecs, vec, sigmas = _chunk(dev, 4)
    for args, message in (((noise, vecs, vec, sigmas[:-1]), "sigmas"), ((noise[:, :100], vecs, vec, sigmas), "noise"),
                          ((noise[..., :128], vecs, vec, sigmas), "noise")):
        with pytest.raises(ValueError, match=message):
            m.generate_chunk(*args)
        assert m.cache_valid_len == 512 and all(a is b for a, b in zip(m.caches, caches))
        assert all(h.length == 512 and torch.equal(h.mass, w) for h, w in zip(m.histories, mass))
    m.generate_chunk(noise, vecs, vec, sigmas)
    assert m.cache_valid_len == 300 + 128


@pytest.mark.parametrize("cap", [140, 2000])
def test_layer_history_moves_to_a_cache_of_another_size(dev, cap):
    """After an eviction into a smaller or larger cache the bounds are that cache's: the
    roll-out goes on to its end."""
    hist, kvc = pkg_module("kv_history"), pkg_module("fp8_kv_cache")
    g = _gen(dev, cap)
    H, L = 2, 100
    cache, out = kvc.make_fp8_kv_block(1, 300, H, D, device=dev), kvc.make_fp8_kv_block(1, cap, H, D, device=dev)
    h = hist.LayerHistory(cache, top_k=3, q_block=32, keep_first=1, keep_last=1, track_mass=True)

    def write(c, kv):
        q, k, v = (torch.randn(1, L, H, D, device=dev, generator=g).to(BF16) for _ in range(3))
        kvc.quantize_kv_pair_into(c, k, v, kv)
        h.attend(q, k, v, c, kv, True)
        h.commit(c)

    for kv in range(0, 300, L):
        write(cache, kv)
    h.evict(cache, out, 300, 40)
    for kv in range(40, cap - L + 1, L):
        write(out, kv)
    end = h.length
    assert end == 40 + (cap - 40) // L * L and h.mass.shape == (1, H, end)
    ref = hist.make_block_bounds(out)
    hist.update_block_bounds(ref, out, 0, end)
    assert torch.equal(h.bounds, ref)
    q, k, v = (torch.randn(1, L, H, D, device=dev, generator=g).to(BF16) for _ in range(3))
    idx = hist.select_blocks(q, ref, end, 3, q_block=32, keep_first=1, keep_last=1) if end > 192 else None
    ref = _attend(q, out, end, idx, 64, 32 if idx is not None else 128, k, v, None, None)
    # (read whole, the dense attention answers, whose probabilities are fp16 as well)
    assert ((h.attend(q, k, v, out, end, False).to(F64) - ref[0]).abs() <= 2 * ref[2]).all()


@pytest.mark.parametrize("kv", [500, 20000])               # without and with key splits
@pytest.mark.parametrize("Lq,q_block", [(4, 1), (20, 20), (50, 50), (100, 100)])
def test_attention_of_nan_rows(dev, Lq, q_block, kv):
    """A query row that meets a NaN gets NaN in its output and its log-sum-exp (zeros and
    -inf say that it had no key); the other rows are what they were."""
    ca = pkg_module("cache_attention")
    g = _gen(dev, 90 + Lq)
    cache = _cache(dev, 1, kv, 2, "fp8", g)
    q = torch.randn(1, Lq, 2, D, device=dev, generator=g).to(BF16)
    n = -(-kv // 64)
    idx = torch.arange(n, dtype=torch.int32, device=dev).expand(1, 2, -(-Lq // q_block), n)
    ref = _attend(q, cache, kv, idx, 64, q_block, None, None, None, None)
    bad = q.clone()
    bad[0, 1, 0, 5] = float("nan")
    bad[0, 2, 1, 7] = INF                                  # logits of both signs: inf - inf
    no = torch.zeros(1, 2, Lq, dtype=torch.bool, device=dev)
    no[0, 0, 1] = no[0, 1, 2] = True
    for lists in (idx, None):
        out, lse = ca.sparse_chunk_attention(bad, cache, kv, lists, q_block=q_block)
        assert torch.equal(torch.isnan(lse), no)
        assert torch.equal(torch.isnan(out).transpose(1, 2), no[..., None].expand(-1, -1, -1, D))
        yes = ~no
        assert ((out.transpose(1, 2)[yes].to(F64) - ref[0].transpose(1, 2)[yes]).abs() <= ref[2].transpose(1, 2)[yes]).all()
        assert ((lse[yes].to(F64) - ref[1][yes]).abs() <= ref[3][yes]).all()
        hist = pkg_module("kv_history")                    # such a row adds nothing to a mass
        gone, without = q.clone(), torch.where(no, -INF, lse)
        gone[0, 1, 0] = gone[0, 2, 1] = 0
        assert torch.equal(hist.key_mass(bad, lse, cache, kv), hist.key_mass(gone, without, cache, kv))


@pytest.mark.parametrize("Lq,q_block", [(3, 1), (20, 20), (50, 50), (100, 100)])
def test_attention_of_small_values(dev, Lq, q_block):
    """V near 2^-20: as fp16 it is a multiple of 2^-24, off by less than one of them toward
    zero, as _attend's bound on the output allows; a run of one row keeps it in fp32."""
    ca = pkg_module("cache_attention")
    g = _gen(dev, 70 + Lq)
    cache = _cache(dev, 1, 900, 2, "int8", g)
    cache["v_scale"].mul_(2.0 ** -20)
    q, k, v = (torch.randn(1, Lq, 2, D, device=dev, generator=g).to(BF16) for _ in range(3))
    v = (v.float() * 2.0 ** -20).to(BF16)
    idx = _lists(dev, 1, 2, -(-Lq // q_block), 15, 9, g)
    ref = _attend(q, cache, 900, idx, 64, q_block, k, v, None, None)
    got = ca.sparse_chunk_attention(q, cache, 900, idx, q_block=q_block, k_cur=k, v_cur=v)
    _check_attention(got, ref, "small values")
    if q_block == 1:
        bound = ref[2] - 2.0 ** -24                        # without the term for V's last place
        assert ((got[0].to(F64) - ref[0]).abs() <= bound).all()


@pytest.mark.parametrize("kv", [500, 20000])
@pytest.mark.parametrize("Lq,q_block", [(4, 1), (20, 20), (50, 50), (100, 100)])
def test_attention_of_a_nan_value(dev, Lq, q_block, kv):
    """A NaN among the values is in the outputs of the head's rows alone: the log-sum-exp is
    the keys'."""
    ca = pkg_module("cache_attention")
    g = _gen(dev, 190 + Lq)
    cache = _cache(dev, 1, kv, 2, "fp8", g)
    q = torch.randn(1, Lq, 2, D, device=dev, generator=g).to(BF16)
    n = -(-kv // 64)
    idx = torch.arange(n, dtype=torch.int32, device=dev).expand(1, 2, -(-Lq // q_block), n)
    ref = _attend(q, cache, kv, idx, 64, q_block, None, None, None, None)
    cache["v_scale"][0, 77, 1] = float("nan")
    for lists in (idx, None):
        out, lse = ca.sparse_chunk_attention(q, cache, kv, lists, q_block=q_block)
        assert torch.isnan(out[:, :, 1]).all()
        assert ((out[:, :, 0].to(F64) - ref[0][:, :, 0]).abs() <= ref[2][:, :, 0]).all()
        assert ((lse.to(F64) - ref[1]).abs() <= ref[3]).all()
