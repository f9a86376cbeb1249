"""The paged KV cache on the GPU: writes against the contiguous cache's codes, attention
against 64 bits, page copies and decodes against indexing, and a run of them together."""
import math

import pytest
import torch

from conftest import pkg_module

pytestmark = pytest.mark.gpu

BF16, F64, I32 = torch.bfloat16, torch.float64, torch.int32
NAMES = ("k", "v", "k_scale", "v_scale")


def _mods():
    return pkg_module("kv_pages"), pkg_module("cache_attention"), pkg_module("fp8_kv_cache")


def _pool(dev, g, pages, page, H, fmt="fp8", layers=None, gain=1.0):
    """A pool of quantized normal values."""
    kp, _, kvc = _mods()
    code = torch.float8_e4m3fn if fmt == "fp8" else torch.int8
    pool = kp.make_pages(pages, H, page=page, layers=layers, code_dtype=code, device=dev)
    make = kvc.make_fp8_kv_block if fmt == "fp8" else kvc.make_int8_kv_block
    for i in range(layers or 1):
        block = make(pages, page, H, 128, device=dev)
        k, v = ((torch.randn(pages, page, H, 128, device=dev, generator=g) * gain).to(BF16) for _ in range(2))
        kvc.quantize_kv_pair_into(block, k, v, 0)
        for n in NAMES:
            (pool[n] if layers is None else pool[n][i]).copy_(block[n])
    return pool


# Tables as wide as their sequences, and with room for many more tokens: which kernel takes
# a call of more than 32 rows depends on it.
rooms = pytest.mark.parametrize("room", [0, 5120])


def _table(dev, g, lens, page, pages, width=None, room=0):
    """Distinct random pages for every sequence, -1 behind its last."""
    need = [-(-n // page) for n in lens]
    t = torch.full((len(lens), max(width or max(1, *need), room // page)), -1, dtype=I32)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(int(g.initial_seed()))).tolist()
    for b, n in enumerate(need):
        t[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=I32)
    return t.to(dev)


def _i32(dev, values):
    return torch.tensor(values, dtype=I32, device=dev)


def _held(pool, key, table, b, n):
    """bf16(code * scale) of the first n tokens of a sequence, in 64 bits."""
    page = pool[key].shape[1]
    t = torch.arange(n, device=table.device)
    pg = table[b].long()[t // page]
    codes = pool[key]
    x = codes.view(torch.uint8)[pg, t % page].view(codes.dtype).float() * pool[key + "_scale"][pg, t % page]
    return x.to(BF16).to(F64)


def _reference(q, pool, table, lens, causal=False, k_cur=None, v_cur=None, cur_valid=None, scale=None,
               first=None):
    """out, lse, the rows' sum of p |v| / sum p, and the largest sum of |q k| scale."""
    B, Lq, Hq, D = q.shape
    H = pool["k"].shape[2]
    G, dev = Hq // H, q.device
    scale = D ** -0.5 if scale is None else scale
    out, spread = torch.zeros(2, B, Lq, Hq, D, dtype=F64, device=dev).unbind(0)
    lse = torch.full((B, Hq, Lq), -math.inf, dtype=F64, device=dev)
    terms = torch.zeros(B, Hq, Lq, dtype=F64, device=dev)
    for b in range(B):
        k, v = _held(pool, "k", table, b, lens[b]), _held(pool, "v", table, b, lens[b])
        seen = torch.ones(Lq, lens[b], dtype=torch.bool, device=dev)
        if causal:
            start = lens[b] - Lq if first is None else first[b]
            seen = torch.arange(lens[b], device=dev) <= start + torch.arange(Lq, device=dev)[:, None]
        if k_cur is not None:
            k, v = torch.cat([k, k_cur[b].to(F64)]), torch.cat([v, v_cur[b].to(F64)])
            ok = torch.ones(k_cur.shape[1], dtype=torch.bool, device=dev) if cur_valid is None else cur_valid[
                b if cur_valid.shape[0] > 1 else 0, :k_cur.shape[1]].bool()
            seen = torch.cat([seen, ok.expand(Lq, -1)], 1)
        v = torch.where(seen.any(0)[:, None, None], v, torch.zeros_like(v)) if len(v) else v
        for h in range(Hq):
            if not len(k):
                continue
            kh, vh, qh = k[:, h // G], v[:, h // G], q[b, :, h].to(F64)
            s = (qh @ kh.T * scale).masked_fill(~seen, -math.inf)
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
            total = p.sum(-1, keepdim=True)
            w = torch.where(total > 0, p / total, torch.zeros_like(p))
            out[b, :, h], spread[b, :, h] = w @ vh, w @ vh.abs()
            lse[b, h] = torch.where(total > 0, top + total.log(), -math.inf)[:, 0]
            terms[b, h] = (qh.abs() @ kh.abs().T * scale).masked_fill(~seen, 0.0).amax(-1)
    return out, lse, spread, terms


def _check(got, want, what=""):
    """Output: half a step of bf16 at the result, and what moves the probabilities: fp16
    (2^-11 relative), the logit's fp32 sum of 128 terms (129 2^-24 of the terms), exp2 and
    the fp32 sums (2^-20). Log-sum-exp: the logit's error, 2^-20, and 2^-22 of itself."""
    out, lse = got
    ref, rlse, spread, terms = want
    assert torch.isfinite(out).all(), what
    logit = 129 * 2.0 ** -24 * terms
    rel = (2.0 ** -11 + 2.0 ** -20 + 2 * logit).transpose(1, 2)[..., None]
    err = rel * spread + 1e-30
    tol = err + (ref.abs() + err) * 2.0 ** -8
    worst = ((out.to(F64) - ref).abs() / tol).max().item() if out.numel() else 0.0
    none = rlse == -math.inf
    assert torch.equal(lse == -math.inf, none), what
    assert (out.transpose(1, 2)[none] == 0).all(), what
    d = (lse.to(F64) - rlse).abs()[~none]
    ltol = (logit + 2.0 ** -20 + rlse.abs() * 2.0 ** -22)[~none]
    lworst = (d / ltol).max().item() if d.numel() else 0.0
    print(f"[pages] {what}: out {worst:.2f} lse {lworst:.2f} of the tolerance", flush=True)
    assert worst <= 1.0 and lworst <= 1.0, (what, worst, lworst)


# --------------------------------------------------------------------------
# attention

@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("H,G", [(8, 4), (3, 1), (1, 16), (2, 17), (1, 40)])
@pytest.mark.parametrize("lens", [(1,), (700, 0, 64, 65, 63, 1), (129, 128, 127), (4111, 33)])
def test_one_token(dev, fmt, H, G, lens):
    _, ca, _ = _mods()
    g = torch.Generator(device=dev).manual_seed(sum(lens) + 7 * H + G)
    pages = sum(-(-n // 64) for n in lens) + 2
    pool = _pool(dev, g, pages, 64, H, fmt)
    table = _table(dev, g, lens, 64, pages)
    q = torch.randn(len(lens), 1, H * G, 128, device=dev, generator=g).to(BF16)
    got = ca.paged_attention(q, pool, table, _i32(dev, lens))
    _check(got, _reference(q, pool, table, lens), f"{fmt} {H}x{G} {lens}")


@rooms
@pytest.mark.parametrize("page", [64, 256, 1024])
@pytest.mark.parametrize("Lq,G", [(2, 1), (5, 4), (8, 2), (9, 4), (33, 1), (70, 3), (129, 1), (300, 1), (101, 5)])
def test_causal(dev, page, Lq, G, room):
    """Sequences shorter than the queries have rows without a key."""
    _, ca, _ = _mods()
    lens = (Lq, 1000, max(1, Lq // 2), 0, 513 + Lq)
    g = torch.Generator(device=dev).manual_seed(page + Lq)
    pages = sum(-(-n // page) for n in lens) + 1
    pool = _pool(dev, g, pages, page, 2)
    table = _table(dev, g, lens, page, pages, room=room)
    q = torch.randn(len(lens), Lq, 2 * G, 128, device=dev, generator=g).to(BF16)
    got = ca.paged_attention(q, pool, table, _i32(dev, lens), causal=True)
    _check(got, _reference(q, pool, table, lens, causal=True), f"page {page} Lq {Lq} G {G}")


@rooms
@pytest.mark.parametrize("Lq,G", [(1, 1), (7, 2), (40, 1), (200, 2)])
def test_causal_queries_of_their_own_places(dev, Lq, G, room):
    """Prompts of different lengths: rows before a sequence's first token see none, rows
    past its last see all of it."""
    _, ca, _ = _mods()
    H, page, lens, first = 2, 64, (700, 230, 64, 5, 0), (700 - Lq // 2, 230 - Lq, 3, -3, 0)
    g = torch.Generator(device=dev).manual_seed(Lq)
    pool = _pool(dev, g, 30, page, H)
    table = _table(dev, g, lens, page, 30, room=room)
    q = torch.randn(len(lens), Lq, H * G, 128, device=dev, generator=g).to(BF16)
    got = ca.paged_attention(q, pool, table, _i32(dev, lens), causal=True, q_start=_i32(dev, first))
    _check(got, _reference(q, pool, table, lens, causal=True, first=first), f"{Lq} rows")
    last = ca.paged_attention(q, pool, table, _i32(dev, lens), causal=True)
    same = ca.paged_attention(q, pool, table, _i32(dev, lens), causal=True, q_start=_i32(dev, [n - Lq for n in lens]))
    assert torch.equal(last[0], same[0]) and torch.equal(last[1], same[1])
    far = ca.paged_attention(q, pool, table, _i32(dev, lens), causal=True, q_start=_i32(dev, [2 ** 31 - 1] * 5))
    _check(far, _reference(q, pool, table, lens), "queries past the end")
    none = ca.paged_attention(q, pool, table, _i32(dev, lens), causal=True, q_start=_i32(dev, [-2 ** 31] * 5))
    assert (none[0] == 0).all() and (none[1] == -math.inf).all()


def test_prompts_of_one_batch(dev):
    """Prompts of different lengths written and attended in one pass: as each alone."""
    kp, _, _ = _mods()
    H, adds = 2, (70, 1, 0, 33)
    g = torch.Generator(device=dev).manual_seed(2)
    cache = kp.PagedKVCache(1, 20, H, page=64, device=dev)
    cache.pool["k"].view(torch.uint8).fill_(0x7f)  # (NaN codes: what no token was written to)
    cache.pool["v"].view(torch.uint8).fill_(0x7f)
    old = torch.randn(4, 100, 2, H, 128, device=dev, generator=g).to(BF16)
    seqs = [cache.new() for _ in adds]
    batch = cache.open(seqs, [100, 64, 3, 0])
    batch.write(0, old[:, :, 0], old[:, :, 1])
    batch.commit()
    q, k, v = torch.randn(4, 70, 3, H, 128, device=dev, generator=g).to(BF16).unbind(2)
    batch = cache.open(seqs, adds)
    batch.write(0, k, v)
    out, lse = batch.attend(0, q, causal=True)
    batch.commit()
    for b, (s, n) in enumerate(zip(seqs, adds)):
        if n:
            one = cache.open([s])
            want = _reference(q[b:b + 1, :n], cache.layer(0), one.table, (cache.length(s),), causal=True)
            _check((out[b:b + 1, :n], lse[b:b + 1, :, :n]), want, f"prompt {b}")


@pytest.mark.parametrize("Lq", [1, 40, 200])
def test_a_pool_without_pages(dev, Lq):
    """No key but the tail's, or none at all."""
    kp, ca, _ = _mods()
    pool = kp.make_pages(0, 2, device=dev)
    table, n = torch.zeros(3, 0, dtype=I32, device=dev), _i32(dev, (0, 5, 70))
    g = torch.Generator(device=dev).manual_seed(Lq)
    q = torch.randn(3, Lq, 2, 128, device=dev, generator=g).to(BF16)
    out, lse = ca.paged_attention(q, pool, table, n)
    assert (out == 0).all() and (lse == -math.inf).all()
    k, v = torch.randn(3, 67, 2, 2, 128, device=dev, generator=g).to(BF16).unbind(2)
    got = ca.paged_attention(q, pool, table, n, k_cur=k, v_cur=v)
    _check(got, _reference(q, pool, table, (0, 0, 0), k_cur=k, v_cur=v), "tail alone")
    wide = ca.paged_attention(q, pool, torch.zeros(3, 4, dtype=I32, device=dev), n, k_cur=k, v_cur=v)
    assert torch.equal(wide[0], got[0]) and torch.equal(wide[1], got[1])
    kp.write_pages(pool, k, v, table, n)
    assert kp.read_pages(pool, "k", table, n, 5).abs().sum().item() == 0


@rooms
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("Lq,G,Lc", [(1, 1, 1), (1, 4, 70), (31, 1, 200), (130, 1, 0), (129, 2, 129), (300, 1, 64), (65, 1, 1)])
@pytest.mark.parametrize("masked", [False, True])
def test_queries_and_tail(dev, fmt, Lq, G, Lc, masked, room):
    """Any number of queries, with the current chunk's keys behind the history, padded
    ones among them, and what a masked key holds without effect."""
    _, ca, _ = _mods()
    lens, page, H = (0, 777, 64, 1301), 128, 2
    g = torch.Generator(device=dev).manual_seed(Lq + G + Lc)
    pages = sum(-(-n // page) for n in lens) + 1
    pool = _pool(dev, g, pages, page, H, fmt)
    table = _table(dev, g, lens, page, pages, room=room)
    B = len(lens)
    q = torch.randn(B, Lq, H * G, 128, device=dev, generator=g).to(BF16)
    kw = {}
    if Lc:
        qkv = torch.randn(B, Lc, 3, H, 128, device=dev, generator=g).to(BF16)
        kw = dict(k_cur=qkv[:, :, 1], v_cur=qkv[:, :, 2])
    if masked and Lc:
        valid = torch.rand(B, Lc, device=dev, generator=g) < 0.7
        valid[0] = False  # no history either: rows without a key
        kw["cur_valid"] = valid
        qkv[:, :, 1:][~valid] = float("nan")
    got = ca.paged_attention(q, pool, table, _i32(dev, lens), **kw)
    if masked and Lc:
        qkv[:, :, 1:][~valid] = 0.0
    _check(got, _reference(q, pool, table, lens, **kw), f"{fmt} Lq {Lq} G {G} Lc {Lc} masked {masked}")


@rooms
@pytest.mark.parametrize("Lq", [1, 9, 40, 200])
def test_what_lies_behind_a_sequence_does_not_matter(dev, Lq, room):
    """NaN codes and infinite scales behind the end, in unnamed pages and under entries
    that name none; such entries inside a sequence name no keys."""
    _, ca, _ = _mods()
    H, page, lens = 2, 64, (300, 65)
    g = torch.Generator(device=dev).manual_seed(Lq)
    pool = _pool(dev, g, 12, page, H)
    table = _table(dev, g, lens, page, 12, width=9, room=room)
    q = torch.randn(2, Lq, H, 128, device=dev, generator=g).to(BF16)
    want = ca.paged_attention(q, pool, table, _i32(dev, lens))
    _check(want, _reference(q, pool, table, lens), "clean")
    used = torch.zeros(12, page, dtype=torch.bool, device=dev)
    for b, n in enumerate(lens):
        t = torch.arange(n, device=dev)
        used[table[b].long()[t // page], t % page] = True
    for key in ("k", "v"):
        pool[key].view(torch.uint8)[~used] = 0x7F
        pool[key + "_scale"][~used] = float("inf")
    table[0, 5:], table[1, 2:] = 2 ** 31 - 1, -2 ** 31
    got = ca.paged_attention(q, pool, table, _i32(dev, lens))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # a hole: its keys are absent, and lengths past the table end with it
    table[0, 1] = 12
    got = ca.paged_attention(q, pool, table, _i32(dev, (2 ** 31 - 1, -5)))
    t = torch.tensor([i for i in range(300) if i // page != 1 and i // page < 5], device=dev)
    mine = table[0, :5].clone()
    mine[1] = 0
    pg = mine.long()[t // page]
    full = {n: x[pg, t % page][None] for n, x in ((n, pool[n].view(torch.uint8) if n in "kv" else pool[n]) for n in NAMES)}
    full["k"], full["v"] = full["k"].view(pool["k"].dtype), full["v"].view(pool["v"].dtype)
    kvc = {n: torch.zeros(1, 1024, *x.shape[2:], dtype=x.dtype, device=dev) for n, x in full.items()}
    for n in NAMES:
        a, b = (x.view(torch.uint8) if n in "kv" else x for x in (kvc[n], full[n]))
        a[:, :len(t)] = b
    # (the last page is whole here: its tokens behind 300 are NaN, so the length stays 300 in the reference)
    got = ca.paged_attention(q, pool, table, _i32(dev, (300, -5)))
    ref = _reference(q[:1], kvc, torch.zeros(1, 1, dtype=I32, device=dev), (len(t),))
    _check((got[0][:1], got[1][:1]), ref, "hole")
    assert (got[0][1] == 0).all() and (got[1][1] == -math.inf).all()


@rooms
@pytest.mark.parametrize("Lq", [1, 40, 150])
def test_nan_and_extreme_logits(dev, Lq, room):
    """A row that meets a NaN gets NaN in output and log-sum-exp; rows of other
    sequences do not. Logits of +-1e4 stay a softmax."""
    _, ca, _ = _mods()
    H, page, lens = 2, 64, (200, 200)
    g = torch.Generator(device=dev).manual_seed(Lq)
    pool = _pool(dev, g, 8, page, H, gain=30.0)
    table = _table(dev, g, lens, page, 8, room=room)
    q = (torch.randn(2, Lq, H, 128, device=dev, generator=g) * 30).to(BF16)
    got = ca.paged_attention(q, pool, table, _i32(dev, lens))
    _check(got, _reference(q, pool, table, lens), "large logits")
    q[0, 0, 0, 5] = float("nan")
    bad = ca.paged_attention(q, pool, table, _i32(dev, lens))
    assert torch.isnan(bad[0][0, 0, 0]).all() and torch.isnan(bad[1][0, 0, 0])
    bad[0][0, 0, 0], bad[1][0, 0, 0] = got[0][0, 0, 0], got[1][0, 0, 0]
    assert torch.equal(bad[0], got[0]) and torch.equal(bad[1], got[1])


def test_strides_scale_and_scratch_of_other_calls(dev):
    """A pool with token-major scales inside a larger one, a q view, a strided table, a
    scale of one's own: as the plain layout."""
    _, ca, _ = _mods()
    H, page, lens = 4, 64, (515, 1024, 3)
    g = torch.Generator(device=dev).manual_seed(5)
    pool = _pool(dev, g, 30, page, H)
    table = _table(dev, g, lens, page, 30)
    q = torch.randn(3, 2, H, 128, device=dev, generator=g).to(BF16)
    want = ca.paged_attention(q, pool, table, _i32(dev, lens), softmax_scale=0.2)
    _check(want, _reference(q, pool, table, lens, scale=0.2), "plain layout")
    other = {}
    for n in NAMES:
        x = pool[n].contiguous()
        wide = torch.zeros(30, page, 2 * H, x.shape[3], dtype=x.dtype, device=dev)
        wide[:, :, H:] = x
        other[n] = wide[:, :, H:]
    qkv = torch.randn(3, 2, 3, H, 128, device=dev, generator=g).to(BF16)
    qkv[:, :, 0] = q
    t2 = torch.stack([table, table], 2)
    got = ca.paged_attention(qkv[:, :, 0], other, t2[:, :, 1], _i32(dev, lens), softmax_scale=0.2)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@rooms
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("Lq,Lc,causal", [(1, 0, False), (9, 0, True), (2, 70, False), (20, 0, True)])
@pytest.mark.parametrize("B,lens", [(70, 130), (150, 40), (300, 40)])
def test_many_sequences(dev, B, lens, Lq, Lc, causal, fmt, room):
    _, ca, _ = _mods()
    n = [(lens * (b + 1) * 7919) % (3 * lens) for b in range(B)]
    g = torch.Generator(device=dev).manual_seed(B)
    pages = sum(-(-x // 64) for x in n) + 1
    pool = _pool(dev, g, pages, 64, 2, fmt)
    table = _table(dev, g, n, 64, pages, room=room)
    q = torch.randn(B, Lq, 4, 128, device=dev, generator=g).to(BF16)
    kw = dict(causal=causal)
    if Lc:
        kv = torch.randn(2, B, Lc, 2, 128, device=dev, generator=g).to(BF16)
        kw.update(k_cur=kv[0], v_cur=kv[1], cur_valid=torch.rand(B, Lc, device=dev, generator=g) < 0.5)
    _check(ca.paged_attention(q, pool, table, _i32(dev, n), **kw), _reference(q, pool, table, n, **kw), f"B {B}")


@pytest.mark.parametrize("Lq", [1, 5, 150])
def test_one_long_sequence(dev, Lq):
    """Every workgroup holds a part of the same few items."""
    _, ca, _ = _mods()
    page, lens = 1024, (100_001,)
    g = torch.Generator(device=dev).manual_seed(Lq)
    pool = _pool(dev, g, 99, page, 1)
    table = _table(dev, g, lens, page, 99)
    q = torch.randn(1, Lq, 3, 128, device=dev, generator=g).to(BF16)
    got = ca.paged_attention(q, pool, table, _i32(dev, lens), causal=True)
    _check(got, _reference(q, pool, table, lens, causal=True), f"{Lq} rows")


def test_offsets_past_32_bits(dev):
    """A pool whose codes pass 4 GiB, its last pages read, written and copied."""
    kp, ca, _ = _mods()
    H, page = 16, 256
    pages = (1 << 32) // (page * H * 128) + 40
    g = torch.Generator(device=dev).manual_seed(3)
    pool = kp.make_pages(pages, H, page=page, device=dev)
    n, first = 5 * page - 30, pages - 6
    table = torch.arange(first, first + 5, dtype=I32, device=dev)[None]
    k, v = (torch.randn(1, n, H, 128, device=dev, generator=g).to(BF16) for _ in range(2))
    kp.write_pages(pool, k, v, table, _i32(dev, [0]))
    q = torch.randn(1, 3, H, 128, device=dev, generator=g).to(BF16)
    tail = {m: pool[m][first:first + 5] for m in NAMES}
    at = torch.arange(5, dtype=I32, device=dev)[None]
    for lq in (1, 3):
        got = ca.paged_attention(q[:, :lq], pool, table, _i32(dev, [n]))
        _check(got, _reference(q[:, :lq], tail, at, (n,)), f"far pages Lq {lq}")
    big = torch.randn(1, 200, H, 128, device=dev, generator=g).to(BF16)
    for room in (0, 10):
        far = torch.nn.functional.pad(table, (0, room), value=-1)
        got = ca.paged_attention(big, pool, far, _i32(dev, [n]))
        _check(got, _reference(big, tail, at, (n,)), "far pages, 200 queries")
    assert torch.equal(kp.read_pages(pool, "k", table, _i32(dev, [n]), n), kp.read_pages(tail, "k", at, _i32(dev, [n]), n))
    kp.copy_pages(pool, [pages - 3], [pages - 1])
    for m in NAMES:
        a, b = (pool[m][e].contiguous().view(torch.uint8) for e in (pages - 3, pages - 1))
        assert torch.equal(a, b)


# --------------------------------------------------------------------------
# write, read, copy

@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("layout", ["bshd", "bhsd", "qkv"])
@pytest.mark.parametrize("L,H", [(1, 1), (1, 8), (1, 70), (3, 24), (64, 5), (129, 24), (1000, 2), (700, 1), (513, 3)])
def test_write_is_the_contiguous_write(dev, fmt, layout, L, H):
    """Codes and scales are the contiguous cache's, token for token; nothing else of the
    pool changes: rows behind the counts, pages of nobody."""
    kp, _, kvc = _mods()
    page, starts = 64, (0, 63, 100)
    counts = (L, max(0, L - 1), L // 2)
    g = torch.Generator(device=dev).manual_seed(L * H)
    if layout == "bshd":
        k, v = (torch.randn(3, L, H, 128, device=dev, generator=g).to(BF16) for _ in range(2))
    elif layout == "bhsd":
        k, v = (torch.randn(3, H, L, 128, device=dev, generator=g).to(BF16).transpose(1, 2) for _ in range(2))
    else:
        qkv = torch.randn(3, L, 3, H, 128, device=dev, generator=g).to(BF16)
        k, v = qkv[:, :, 1], qkv[:, :, 2]
    k[0, 0, 0] = 0.0  # a row of zeros: scale 1
    if L > 1:
        k[2, -1] = float("nan")  # behind the counts
    make = kvc.make_fp8_kv_block if fmt == "fp8" else kvc.make_int8_kv_block
    flat = make(3, 100 + L, H, 128, device=dev)
    for b in range(3):
        one = {n: x[b:b + 1] for n, x in flat.items()}
        kvc.quantize_kv_pair_into(one, k[b:b + 1, :counts[b]], v[b:b + 1, :counts[b]], starts[b])
    ends = [s + c for s, c in zip(starts, counts)]
    pages = sum(-(-e // page) for e in ends) + 2
    pool = _pool(dev, g, pages, page, H, fmt)
    before = {n: x.clone() for n, x in pool.items()}
    table = _table(dev, g, ends, page, pages)
    status = torch.full((1,), 7, dtype=I32, device=dev)
    kp.write_pages(pool, k, v, table, _i32(dev, starts), counts=_i32(dev, counts), status=status)
    assert status.item() == 0
    for n in NAMES:
        want, got = before[n], pool[n]
        raw = (lambda x: x.view(torch.uint8)) if n in "kv" else (lambda x: x)
        for b in range(3):
            t = torch.arange(starts[b], ends[b], device=dev)
            raw(want)[table[b].long()[t // page], t % page] = raw(flat[n])[b, starts[b]:ends[b]]
        assert torch.equal(raw(want), raw(got)), n


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("L", [1, 200])
def test_scales_of_a_torch_program(dev, fmt, L):
    """gpu_scales: amax / 448.0 (127.0) and the codes of it as torch computes them on the
    GPU, bit for bit; rows of every magnitude, zeros and the largest values among them."""
    kp, _, _ = _mods()
    g = torch.Generator(device=dev).manual_seed(L)
    kv = [torch.randn(2, L, 24, 128, device=dev, generator=g) for _ in range(2)]
    for x in kv:
        x *= torch.exp2(torch.randint(-126, 126, (2, L, 24, 1), device=dev, generator=g).float())
        x[0, 0, 0] = 0.0
        x[1, 0, 1] = torch.finfo(BF16).max
    kv = [x.to(BF16) for x in kv]
    pages = 2 * -(-L // 64)
    pool = _pool(dev, g, pages, 64, 24, fmt)
    table = torch.arange(pages, dtype=I32, device=dev).view(2, -1)
    kp.write_pages(pool, *kv, table, _i32(dev, [0, 0]), gpu_scales=True)
    for key, x in zip("kv", kv):
        x = x.float()
        amax = x.abs().amax(-1, keepdim=True)
        s = torch.where(amax > 0, amax / (448.0 if fmt == "fp8" else 127.0), torch.ones_like(amax))
        y = x / s
        codes = y.to(torch.float8_e4m3fn) if fmt == "fp8" else torch.where(
            y >= 0, torch.floor(y + 0.5), torch.ceil(y - 0.5)).clamp(-127, 127).to(torch.int8)
        t = torch.arange(L, device=dev)
        for b in range(2):
            at = table[b].long()[t // 64], t % 64
            assert torch.equal(pool[key + "_scale"][at], s[b])
            assert torch.equal(pool[key].view(torch.uint8)[at], codes[b].view(torch.uint8))


@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("B,L", [(2, 3), (3, 700), (1, 33000)])
def test_a_write_of_a_bad_value_writes_nothing(dev, where, value, B, L):
    kp, _, _ = _mods()
    g = torch.Generator(device=dev).manual_seed(1)
    pages = B * -(-L // 64)
    pool = _pool(dev, g, pages, 64, 4)
    before = {n: x.clone() for n, x in pool.items()}
    table = torch.arange(pages, dtype=I32, device=dev).view(B, -1)
    kv = {n: torch.randn(B, L, 4, 128, device=dev, generator=g).to(BF16) for n in "kv"}
    kv[where][B - 1, L - 1, 3, 127] = value
    start = _i32(dev, [0] * B)
    status = torch.zeros(1, dtype=I32, device=dev)
    kp.write_pages(pool, kv["k"], kv["v"], table, start, status=status)
    assert status.item() == 1
    with pytest.raises(ValueError, match="non-finite"):
        kp.write_pages(pool, kv["k"], kv["v"], table, start)
    for n in NAMES:
        a, b = (x.view(torch.uint8) if n in "kv" else x for x in (pool[n], before[n]))
        assert torch.equal(a, b)
    kv[where][B - 1, L - 1, 3, 127] = 1.0
    kp.write_pages(pool, kv["k"], kv["v"], table, start, status=status)
    assert status.item() == 0


@pytest.mark.parametrize("counts", [(300, 0), (0, 300), (0, 0), (1, 300)])
def test_the_status_of_padded_writes(dev, counts):
    """The status stands for the rows that count, whichever those are, after any before it."""
    kp, _, _ = _mods()
    g = torch.Generator(device=dev).manual_seed(3)
    pool = _pool(dev, g, 10, 64, 4)
    table = torch.arange(10, dtype=I32, device=dev).view(2, 5)
    k, v = (torch.randn(2, 300, 4, 128, device=dev, generator=g).to(BF16) for _ in range(2))
    n, start = _i32(dev, counts), _i32(dev, (0, 0))
    for b, c in enumerate(counts):
        k[b, c:], v[b, c:] = float("nan"), float("inf")
    for was in (0, 1, 7):
        status = _i32(dev, [was])
        kp.write_pages(pool, k, v, table, start, counts=n, status=status)
        assert status.item() == 0
    held = kp.read_pages(pool, "k", table, n, 300)
    for b, c in enumerate(counts):
        assert ((held[b, :c].float() - k[b, :c].float()).abs() <= k[b, :c].float().abs().amax(-1, keepdim=True) / 16).all()
        if c:
            bad = k.clone()
            bad[b, c - 1, 0, 0] = float("inf")
            kp.write_pages(pool, bad, v, table, start, counts=n, status=status)
            assert status.item() == 1


def test_tokens_without_a_page_are_dropped(dev):
    """Entries outside the pool, positions past the table, a negative start."""
    kp, _, _ = _mods()
    g = torch.Generator(device=dev).manual_seed(2)
    pool = _pool(dev, g, 4, 64, 2)
    before = {n: x.clone() for n, x in pool.items()}
    table = _i32(dev, [[0, 4], [-1, -7], [2 ** 31 - 1, 1], [2, 3]])
    k, v = (torch.randn(4, 70, 2, 128, device=dev, generator=g).to(BF16) for _ in range(2))
    kp.write_pages(pool, k, v, table, _i32(dev, [0, 0, 64, -1]), assume_finite=True)
    ref = _pool(dev, torch.Generator(device=dev).manual_seed(2), 4, 64, 2)
    kp.write_pages(ref, k[:1, :64], v[:1, :64], _i32(dev, [[0]]), _i32(dev, [0]))
    kp.write_pages(ref, k[2:3, :64], v[2:3, :64], _i32(dev, [[1]]), _i32(dev, [0]))
    for n in NAMES:
        a, b, c = (x.view(torch.uint8) if n in "kv" else x for x in (pool[n], ref[n], before[n]))
        assert torch.equal(a, b) and torch.equal(a[2:], c[2:])
    kp.write_pages(pool, k, v, table, _i32(dev, [2 ** 31 - 1] * 4), assume_finite=True)
    kp.write_pages(pool, k, v, table[:, :0], _i32(dev, [0] * 4), assume_finite=True)
    for n in NAMES:
        a, b = (x.view(torch.uint8) if n in "kv" else x for x in (pool[n], ref[n]))
        assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("H,page,lens,n", [(3, 64, (0, 1, 200), 200), (8, 256, (700, 9), 1000), (1, 1024, (5,), 3), (2, 64, (64,), 0), (2, 64, (1000, 77), 901), (4, 64, (300,), 333)])
def test_read(dev, fmt, H, page, lens, n):
    kp, _, _ = _mods()
    g = torch.Generator(device=dev).manual_seed(n)
    pages = sum(-(-x // page) for x in lens) + 1
    pool = _pool(dev, g, pages, page, H, fmt)
    table = _table(dev, g, lens, page, pages)
    for key in ("k", "v"):
        got = kp.read_pages(pool, key, table, _i32(dev, lens), n)
        assert got.shape == (len(lens), n, H, 128)
        for b, x in enumerate(lens):
            m = min(x, n)
            assert torch.equal(got[b, :m].to(F64), _held(pool, key, table, b, m)) and (got[b, m:] == 0).all()


@pytest.mark.parametrize("layers,page,H,pairs", [(None, 64, 3, 1), (3, 64, 24, 5), (2, 1024, 1, 7), (1, 64, 1, 600)])
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_copy(dev, layers, page, H, pairs, fmt):
    kp, _, _ = _mods()
    g = torch.Generator(device=dev).manual_seed(pairs)
    P = 2 * pairs + 3
    pool = _pool(dev, g, P, page, H, fmt, layers=layers)
    before = {n: x.clone() for n, x in pool.items()}
    order = torch.randperm(P).tolist()
    dst, src = order[:pairs], [order[pairs + i // 2] for i in range(pairs)]  # (one page to two)
    kp.copy_pages(pool, src, dst)
    for n in NAMES:
        want, got = (x.view(torch.uint8) if n in "kv" else x for x in (before[n], pool[n]))
        dim = 0 if layers is None else 1
        want = want.clone().index_copy(dim, torch.tensor(dst, device=dev), want.index_select(dim, torch.tensor(src, device=dev)))
        assert torch.equal(got, want), n


# --------------------------------------------------------------------------
# streams, graphs

def test_captured_calls_follow_the_tables(dev):
    """Write and attention captured once, replayed while lengths, tables and values
    change; two captured graphs beside eager work."""
    kp, ca, _ = _mods()
    H, page, B = 4, 64, 3
    g = torch.Generator(device=dev).manual_seed(9)
    pool = _pool(dev, g, 60, page, H)
    table = torch.full((B, 16), -1, dtype=I32, device=dev)
    start, lens = torch.zeros(2, B, dtype=I32, device=dev).unbind(0)
    k, v = (torch.zeros(B, 1, H, 128, dtype=BF16, device=dev) for _ in range(2))
    q = torch.zeros(B, 1, 2 * H, 128, dtype=BF16, device=dev)
    status = torch.zeros(1, dtype=I32, device=dev)

    def step():
        kp.write_pages(pool, k, v, table, start, status=status)
        return ca.paged_attention(q, pool, table, lens)

    step()
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for _ in range(2):
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(step())
        graphs.append(graph)
    pages = torch.randperm(60)[:48].view(B, 16).to(I32)
    for i, n in enumerate([(0, 5, 900), (1, 64, 127), (700, 1000, 3), (63, 0, 511)]):
        now = torch.Generator(device=dev).manual_seed(i)
        table.copy_(pages.roll(i, 0))
        start.copy_(_i32(dev, n))
        lens.copy_(start + 1)
        for x in (k, v, q):
            x.copy_(torch.randn(x.shape, device=dev, generator=now).to(BF16))
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        out, lse = (x.clone() for x in outs[i % 2])
        eager = step()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[0]) and torch.equal(lse, eager[1]) and status.item() == 0
        _check((out, lse), _reference(q, pool, table, [x + 1 for x in n]), f"replay {i}")


@rooms
@pytest.mark.parametrize("B,Lq,causal", [(2, 1, False), (2, 40, True), (2, 300, True), (2, 300, False), (150, 1, False), (1, 3, True)])
def test_every_kernel_captured(dev, B, Lq, causal, room):
    """One captured call, replayed over other lengths and tables with eager calls between."""
    _, ca, _ = _mods()
    H, page, width = 2, 64, max(13, room // 64)
    g = torch.Generator(device=dev).manual_seed(B + Lq)
    pool = _pool(dev, g, 13 * B, page, H)
    table = torch.full((B, width), -1, dtype=I32, device=dev)
    lens = torch.zeros(B, dtype=I32, device=dev)
    q = torch.randn(B, Lq, 2 * H, 128, device=dev, generator=g).to(BF16)
    call = lambda: ca.paged_attention(q, pool, table, lens, causal=causal)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = call()
    for i in range(4):
        table[:, :13] = torch.randperm(13 * B, generator=torch.Generator().manual_seed(i)).view(B, 13).to(dev, I32)
        lens.copy_(torch.randint(0, 13 * page + 1, (B,), generator=torch.Generator().manual_seed(i)))
        graph.replay()
        got = out.clone(), lse.clone()
        eager = call()
        torch.cuda.synchronize()
        assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1])
        if i == 3:
            _check(got, _reference(q, pool, table, lens.tolist(), causal=causal), f"B {B} Lq {Lq}")


def test_calls_on_two_streams(dev):
    _, ca, _ = _mods()
    H, page, lens = 2, 64, (3000, 2000)
    g = torch.Generator(device=dev).manual_seed(4)
    pages = sum(-(-n // page) for n in lens) + 1
    pool = _pool(dev, g, pages, page, H)
    table, n = _table(dev, g, lens, page, pages), _i32(dev, lens)
    qs = [torch.randn(2, lq, H, 128, device=dev, generator=g).to(BF16) for lq in (1, 1, 40, 150)]
    want = [ca.paged_attention(q, pool, table, n) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    got = []
    for q, s in zip(qs, streams):
        with torch.cuda.stream(s):
            got.append([ca.paged_attention(q, pool, table, n) for _ in range(3)])
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        for x in gs:
            assert torch.equal(x[0], w[0]) and torch.equal(x[1], w[1])


# --------------------------------------------------------------------------
# a run of them together: branches of the AR model

def _model(dev, pages, **kw):
    db = pkg_module("dit_block")
    return db.FP8ARModel(2, 256, 2, (2, 5, 9), 4, device=dev, seed=3, pages=pages, **kw)


def _inputs(dev, model, B, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    noise = torch.randn(B, model.tokens_per_chunk, 256, device=dev, generator=g).to(BF16)
    vecs = [torch.randn(B, 256, device=dev, generator=g).to(BF16) for _ in range(3)]
    return noise, vecs[:2], vecs[2], [1.0, 0.5, 0.0]


def _rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


def test_a_branch_is_a_roll_out_of_the_contiguous_model(dev):
    """Chunk after chunk as the model with one cache a layer. The two attend in another
    order of tiles, so outputs agree to the bf16 steps of a block (2^-8 each, of about ten
    tensor operations a pass, two passes a chunk), the first layer's cache to the codes of
    the first chunk."""
    plain, paged = _model(dev, 0), _model(dev, 9)
    branch = paged.start_branch()
    for i in range(3):
        args = _inputs(dev, plain, 1, i)
        a, b = plain.generate_chunk(*args), paged.generate_chunk(*args, branches=[branch])
        assert _rel(b, a) < 20 * 2.0 ** -8
    assert paged.paged.length(branch) == plain.cache_valid_len == 270
    kp, _, kvc = _mods()
    batch = paged.paged.open([branch])
    for layer in range(2):
        for key in ("k", "v"):
            got = kp.read_pages(paged.paged.layer(layer), key, batch.table, batch.start, 270)
            want = kvc.dequantize_kv(plain.caches[layer], key, 270)
            assert _rel(got, want) < 0.1
            if layer == 0:
                assert _rel(got[:, :90], want[:, :90]) < 20 * 2.0 ** -8


def test_forked_branches(dev):
    """Two branches of one history: equal inputs give equal chunks, other inputs leave the
    origin as it was, and a branch goes on as its origin would have."""
    kp, _, _ = _mods()
    m = _model(dev, 20)
    a = m.start_branch()
    noise, vecs, write, sig = _inputs(dev, m, 1, 0)
    m.generate_chunk(noise, vecs, write, sig, branches=[a])
    b, c = m.fork_branch(a), m.fork_branch(a)
    assert m.paged.free_pages == 18  # 90 tokens: two pages

    def held(branch):
        batch = m.paged.open([branch])
        return [kp.read_pages(m.paged.layer(i), key, batch.table, batch.start, m.paged.length(branch))
                for i in range(2) for key in ("k", "v")]

    origin = held(c)
    two = [torch.cat([x, x]) for x in (noise, *vecs, write)]
    out = m.generate_chunk(two[0], two[1:3], two[3], sig, branches=[a, b])
    assert torch.equal(out[0], out[1])
    assert all(torch.equal(x, y) for x, y in zip(held(a), held(b)))
    args = _inputs(dev, m, 2, 5)
    out = m.generate_chunk(*args, branches=[b, a])
    assert not torch.equal(out[0], out[1])
    assert all(torch.equal(x, y) for x, y in zip(held(c), origin))
    with pytest.raises(ValueError, match="of one length"):
        m.generate_chunk(*_inputs(dev, m, 2, 6), branches=[a, c])
    m.drop_branch(b)
    late = m.generate_chunk(noise, vecs, write, sig, branches=[c])
    again = m.generate_chunk(noise, vecs, write, sig, branches=[m.start_branch()])
    assert late.shape == again.shape
    assert all(torch.equal(x[:, :90], y) for x, y in zip(held(c), origin))
    m.paged.compact()
    assert all(torch.equal(x[:, :90], y) for x, y in zip(held(c), origin))


def test_a_full_pool_and_a_bad_chunk_leave_the_branches(dev):
    m = _model(dev, 3)
    a = m.start_branch()
    args = _inputs(dev, m, 1, 0)
    m.generate_chunk(*args, branches=[a])
    fork = m.fork_branch(a)
    with pytest.raises(ValueError, match="2 pages are needed, 1 are free"):  # (the half page is shared)
        m.generate_chunk(*args, branches=[fork])
    m.drop_branch(fork)
    noise = args[0].clone()
    noise[0, 3, 7] = float("nan")
    with pytest.raises(ValueError, match="non-finite"):
        m.generate_chunk(noise, *args[1:], branches=[a])
    assert m.paged.length(a) == 90 and m.branch_frames[a] == 2 and m.paged.free_pages == 1
    with pytest.raises(ValueError, match="noise must"):
        m.generate_chunk(noise[:, :5], *args[1:], branches=[a])
    with pytest.raises(ValueError, match="distinct"):
        m.generate_chunk(torch.cat([noise, noise]), *args[1:], branches=[a, a])
    with pytest.raises(ValueError, match="no sequence"):
        m.generate_chunk(noise, *args[1:], branches=[99])


def test_drafted_tokens(dev):
    """Five drafted tokens written and attended causally, two accepted: what follows is as
    if the others had never been."""
    kp, ca, _ = _mods()
    cache = kp.PagedKVCache(1, 40, 4, page=64, device=dev)
    g = torch.Generator(device=dev).manual_seed(0)

    def tokens(B, L):
        return torch.randn(B, L, 3, 4, 128, device=dev, generator=g).to(BF16).unbind(2)

    seqs = [cache.new(), cache.new()]
    batch = cache.open(seqs, [300, 63])
    _, k, v = tokens(2, 300)
    batch.write(0, k, v)
    batch.commit()
    batch = cache.open(seqs, 5)
    q, k, v = tokens(2, 5)
    batch.write(0, k, v)
    got = batch.attend(0, q, causal=True)
    _check(got, _reference(q, cache.layer(0), batch.table, (305, 68), causal=True), "drafted")
    batch.commit()
    for s, n in zip(seqs, (302, 65)):
        cache.truncate(s, n)
    one = cache.open(seqs, 1)
    q1, k1, v1 = tokens(2, 1)
    one.write(0, k1, v1)
    out = one.attend(0, q1)
    one.commit()
    fresh = kp.PagedKVCache(1, 40, 4, page=64, device=dev)
    ids = [fresh.new(), fresh.new()]
    for b, (s, n) in enumerate(zip(ids, (302, 65))):
        batch = fresh.open([s], n)
        mine = [kp.read_pages(cache.layer(0), key, one.table[b:b + 1], _i32(dev, [n]), n) for key in ("k", "v")]
        batch.write(0, *mine)  # (decoded values: their codes are the same again)
        batch.commit()
    batch = fresh.open(ids, 1)
    batch.write(0, k1, v1)
    again = batch.attend(0, q1)
    assert torch.equal(out[0], again[0]) and torch.equal(out[1], again[1])


# --------------------------------------------------------------------------
# padded batches

@rooms
@pytest.mark.parametrize("adds,rows", [((7, 5), 16), ((40, 0, 3), 100), ((70, 64), 128), ((129, 200, 1), 256)])
def test_rows_padded_past_the_longest_addition(dev, adds, rows, room):
    """Writes and causal queries of more rows than any sequence adds: each sequence's rows as
    alone, whatever the padding holds (few rows, the 4-wave tiles, the 8-wave ones)."""
    kp, _, _ = _mods()
    H, G, B = 2, 2, len(adds)
    g = torch.Generator(device=dev).manual_seed(rows)
    cache = kp.PagedKVCache(1, 40 + B * (room // 64), H, page=64, device=dev)
    seqs = [cache.new() for _ in adds]
    old = [50 + 37 * b + room // 2 for b in range(B)]
    batch = cache.open(seqs, old)
    k, v = torch.randn(2, B, max(old), H, 128, device=dev, generator=g).to(BF16)
    batch.write(0, k, v)
    batch.commit()
    batch = cache.open(seqs, adds)
    k, v = torch.randn(2, B, rows, H, 128, device=dev, generator=g).to(BF16)
    q = torch.randn(B, rows, H * G, 128, device=dev, generator=g).to(BF16)
    for b, n in enumerate(adds):
        k[b, n:], v[b, n:] = float("nan"), float("inf")
    batch.write(0, k, v)
    out, lse = batch.attend(0, q, causal=True)
    batch.commit()
    for b, (s, n) in enumerate(zip(seqs, adds)):
        one = cache.open([s])
        assert cache.length(s) == old[b] + n
        want = _reference(q[b:b + 1], cache.layer(0), one.table, (old[b] + n,), causal=True, first=(old[b],))
        _check((out[b:b + 1], lse[b:b + 1]), want, f"adds {adds}, sequence {b}")


def test_a_pass_opened_before_a_capture(dev):
    """open and compact are refused inside a capture, which goes on; write and attend of a
    batch from before it replay over new values."""
    kp, _, _ = _mods()
    H = 2
    g = torch.Generator(device=dev).manual_seed(8)
    cache = kp.PagedKVCache(1, 12, H, page=64, device=dev)
    seqs = [cache.new(), cache.new()]
    k, v = torch.randn(2, 2, 100, H, 128, device=dev, generator=g).to(BF16)
    batch = cache.open(seqs, [100, 64])
    batch.write(0, k, v)
    batch.commit()
    batch = cache.open(seqs, 3)
    q, k, v = torch.randn(3, 2, 3, H, 128, device=dev, generator=g).to(BF16)
    status = torch.zeros(1, dtype=I32, device=dev)

    def step():
        batch.write(0, k, v, status=status)
        return batch.attend(0, q, causal=True)

    step()
    graph, free = torch.cuda.CUDAGraph(), cache.free_pages
    with torch.cuda.graph(graph):
        for call in (lambda: cache.open(seqs, 1), cache.compact):
            with pytest.raises(RuntimeError, match="captured"):
                call()
        out, lse = step()
    assert cache.free_pages == free
    for i in range(3):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device=dev, generator=g).to(BF16))
        graph.replay()
        got = out.clone(), lse.clone()
        eager = step()
        assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1]) and status.item() == 0
    _check(got, _reference(q, cache.layer(0), batch.table, (103, 67), causal=True), "replayed")
    batch.commit()


# --------------------------------------------------------------------------
# what is not finite, and causal rows before it

def _before_and_after(fmt, Lq, G, room, dev):
    _, ca, _ = _mods()
    H, page, lens = 2, 64, (700, 230)
    g = torch.Generator(device=dev).manual_seed(Lq + G)
    pool = _pool(dev, g, 20, page, H, fmt)
    table = _table(dev, g, lens, page, 20, room=room)
    q = torch.randn(2, Lq, H * G, 128, device=dev, generator=g).to(BF16)
    at = max(1, Lq // 2)  # the row from which on sequence 0's special token is seen
    place = lens[0] - Lq + at
    where = table[0, place // page].item(), place % page, 1
    return ca, pool, table, q, lens, at, where


few_and_tiles = pytest.mark.parametrize("Lq,G", [(8, 1), (9, 3), (40, 1), (70, 1), (33, 5), (300, 1)])


@rooms
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@few_and_tiles
def test_a_nan_key_reaches_the_rows_that_see_it(dev, fmt, Lq, G, room):
    """NaN in both outputs of those rows and that cached head, no other row differs."""
    ca, pool, table, q, lens, at, where = _before_and_after(fmt, Lq, G, room, dev)
    want = _reference(q, pool, table, lens, causal=True)
    pool["k_scale"][where] = float("nan")
    out, lse = ca.paged_attention(q, pool, table, _i32(dev, lens), causal=True)
    assert torch.isnan(out[0, at:, G:]).all() and torch.isnan(lse[0, G:, at:]).all()
    out[0, at:, G:], lse[0, G:, at:] = want[0][0, at:, G:].to(BF16), want[1][0, G:, at:].float()
    _check((out, lse), want, f"{fmt} Lq {Lq} G {G}")


@rooms
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@few_and_tiles
def test_values_that_causal_rows_do_not_see(dev, fmt, Lq, G, room):
    """A finite V, past fp16's range too, has no part in the rows before its token. A NaN one
    makes the outputs NaN of the rows that see it; the log-sum-exp is the keys' alone."""
    ca, pool, table, q, lens, at, where = _before_and_after(fmt, Lq, G, room, dev)
    want = _reference(q, pool, table, lens, causal=True)
    n = _i32(dev, lens)
    for big in (70000.0, 1e30, 3e38):
        pool["v_scale"][where] = big / (448 if fmt == "fp8" else 127)
        out, lse = ca.paged_attention(q, pool, table, n, causal=True)
        out[0, at:, G:] = want[0][0, at:, G:].to(BF16)  # (rows that see it have sums of their own range)
        _check((out, lse), want, f"V {big}, {fmt} Lq {Lq} G {G}")
    for bad in (float("nan"), float("inf")):
        pool["v_scale"][where] = bad
        out, lse = ca.paged_attention(q, pool, table, n, causal=True)
        seen = out[0, at:, G:]
        assert (torch.isnan(seen) if bad != bad else ~torch.isfinite(seen)).all()
        out[0, :, G:] = want[0][0, :, G:].to(BF16)
        _check((out, lse), want, f"V {bad}, {fmt} Lq {Lq} G {G}")


# --------------------------------------------------------------------------
# instances and promises that the tests above leave open

@rooms
@pytest.mark.parametrize("page", [64, 256])
@pytest.mark.parametrize("Lq,G", [(5, 4), (9, 4), (33, 1), (70, 3), (129, 1), (300, 1), (101, 5)])
def test_causal_int8(dev, page, Lq, G, room):
    _, ca, _ = _mods()
    lens = (Lq, 1000, max(1, Lq // 2), 0, 513 + Lq)
    g = torch.Generator(device=dev).manual_seed(page + Lq)
    pages = sum(-(-n // page) for n in lens) + 1
    pool = _pool(dev, g, pages, page, 2, "int8")
    table = _table(dev, g, lens, page, pages, room=room)
    q = torch.randn(len(lens), Lq, 2 * G, 128, device=dev, generator=g).to(BF16)
    got = ca.paged_attention(q, pool, table, _i32(dev, lens), causal=True)
    _check(got, _reference(q, pool, table, lens, causal=True), f"page {page} Lq {Lq} G {G}")


@rooms
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("B,Lq,Lc,masked,causal", [(2, 1, 70, True, False), (2, 20, 0, False, True), (2, 40, 65, False, False),
                                                   (2, 40, 65, True, False), (2, 300, 65, False, False),
                                                   (2, 300, 65, True, False), (2, 300, 0, False, True),
                                                   (150, 1, 3, True, False), (150, 16, 0, False, True)])
def test_tails_and_formats_captured(dev, fmt, B, Lq, Lc, masked, causal, room):
    """One captured call of each form, replayed over other lengths, tables and masks with eager
    calls between."""
    _, ca, _ = _mods()
    H, page, width = 2, 64, max(13, room // 64)
    g = torch.Generator(device=dev).manual_seed(B + Lq + Lc)
    pool = _pool(dev, g, 13 * B, page, H, fmt)
    table = torch.full((B, width), -1, dtype=I32, device=dev)
    lens = torch.zeros(B, dtype=I32, device=dev)
    q = torch.randn(B, Lq, 2 * H, 128, device=dev, generator=g).to(BF16)
    kw = dict(causal=causal)
    if Lc:
        kv = torch.randn(2, B, Lc, H, 128, device=dev, generator=g).to(BF16)
        kw.update(k_cur=kv[0], v_cur=kv[1])
    if masked:
        kw["cur_valid"] = torch.ones(B, Lc, dtype=torch.bool, device=dev)
    call = lambda: ca.paged_attention(q, pool, table, lens, **kw)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = call()
    for i in range(3):
        now = torch.Generator().manual_seed(i)
        table[:, :13] = torch.randperm(13 * B, generator=now).view(B, 13).to(dev, I32)
        lens.copy_(torch.randint(0, 13 * page + 1, (B,), generator=now))
        if masked:
            kw["cur_valid"].copy_(torch.rand(B, Lc, generator=now) < 0.6)
        graph.replay()
        got = out.clone(), lse.clone()
        eager = call()
        torch.cuda.synchronize()
        assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1])
    if B < 10:
        _check(got, _reference(q, pool, table, lens.tolist(), **kw), f"{fmt} Lq {Lq} Lc {Lc}")


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("Lq,G,room", [(1, 1, 0), (1, 16, 5120), (4, 8, 0), (4, 8, 5120), (1, 64, 5120), (64, 1, 5120)])
def test_probabilities_of_few_rows(dev, fmt, Lq, G, room):
    """Two or a few keys of nearly equal weight whose values cancel: what the probabilities'
    rounding leaves is the output. They are held to 2^-17 of themselves (two bf16); beside it
    the logit's fp32 sum of 128 terms, exp2 and the sums (2^-20), and half a step of bf16 at
    the result. One bf16 would be far off."""
    _, ca, _ = _mods()
    H, page, lens = 2, 64, (2, 8, 34, 300)
    B = len(lens)
    g = torch.Generator(device=dev).manual_seed(Lq + G)
    pool = _pool(dev, g, 9, page, H, fmt)
    for n in ("v", "v_scale"):  # odd tokens: the values of the one before, negated
        pool[n][:, 1::2] = pool[n][:, ::2]
    pool["v_scale"][:, 1::2] *= -1
    table = _table(dev, g, lens, page, 9, room=room)
    q = (torch.randn(B, Lq, H * G, 128, device=dev, generator=g) * 0.05).to(BF16)
    out, lse = ca.paged_attention(q, pool, table, _i32(dev, lens))
    ref, rlse, spread, terms = _reference(q, pool, table, lens)
    rel = (2.0 ** -17 + 2.0 ** -20 + 2 * 129 * 2.0 ** -24 * terms).transpose(1, 2)[..., None]
    tol = rel * spread + (ref.abs() + rel * spread) * 2.0 ** -8 + 1e-30  # (values whose codes are 0: exactly 0)
    worst = ((out.to(F64) - ref).abs() / tol).max().item()
    print(f"[pages] probabilities {fmt} Lq {Lq} G {G}: {worst:.2f} of the tolerance", flush=True)
    assert worst <= 1.0
    assert ((lse.to(F64) - rlse).abs() <= 129 * 2.0 ** -24 * terms + 2.0 ** -20 + rlse.abs() * 2.0 ** -22).all()
    off = 0.0  # (the tolerance tells one bf16 from two)
    for b, n in enumerate(lens):
        k, v = (_held(pool, key, table, b, n) for key in "kv")
        for h in range(H * G):
            s = q[b, :, h].to(F64) @ k[:, h // G].T * 128 ** -0.5
            p = torch.exp(s - s.amax(-1, keepdim=True))
            once = (p.to(BF16).to(F64) @ v[:, h // G]) / p.sum(-1, keepdim=True)
            off = max(off, ((once - ref[b, :, h]).abs() / tol[b, :, h]).max().item())
    assert off > 1.0, off


def test_compiled_calls(dev):
    """torch.compile keeps each op as one node; the registered ops, and calls that a profiler
    sees, are the eager ones."""
    kp, ca, _ = _mods()
    H, page = 2, 64
    g = torch.Generator(device=dev).manual_seed(11)
    pool = _pool(dev, g, 8, page, H)
    table = _i32(dev, [[0, 1, 2], [3, 4, 5]])
    start, lens = _i32(dev, [5, 70]), _i32(dev, [15, 80])
    q, k, v = torch.randn(3, 2, 10, H, 128, device=dev, generator=g).to(BF16)
    status = torch.zeros(1, dtype=I32, device=dev)

    def step(pool, q, k, v):
        kp.write_pages(pool, k, v, table, start, status=status)
        kp.copy_pages(pool, [1, 4], [6, 7])
        out, lse = ca.paged_attention(q, pool, table, lens, causal=True, q_start=start)
        tail, _ = ca.paged_attention(q, pool, table, start, k_cur=k, v_cur=v)
        return out, lse, tail, kp.read_pages(pool, "v", table, lens, 90)

    pools = [{n: t.clone() for n, t in pool.items()} for _ in range(3)]
    eager = step(pools[0], q, k, v)
    compiled = torch.compile(step, backend="aot_eager", fullgraph=True)(pools[1], q, k, v)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        seen = step(pools[2], q, k, v)
    names = {e.key for e in prof.key_averages()}
    assert {"hy_nomas_amd::" + n for n in ("kv_pages_write_", "kv_pages_copy_", "attn_kv_pages", "kv_pages_read")} <= names
    for got, cache in ((compiled, pools[1]), (seen, pools[2])):
        assert all(torch.equal(a, b) for a, b in zip(got, eager))
        for n in NAMES:
            a, b = (x.view(torch.uint8) if n in "kv" else x for x in (cache[n], pools[0][n]))
            assert torch.equal(a, b)


@rooms
@pytest.mark.parametrize("Lq", [1, 20, 40, 300])
def test_masks_tables_and_queries_of_many_shapes(dev, Lq, room):
    """One mask for all sequences, wider than the tail, of bytes; one table row for all; every
    sequence's queries the same memory; a table that is part of a wider one."""
    _, ca, _ = _mods()
    H, page, lens, Lc = 2, 64, (300, 77, 0), 70
    g = torch.Generator(device=dev).manual_seed(Lq)
    pool = _pool(dev, g, 6, page, H)
    row = torch.full((1, 9 + room // page), -1, dtype=I32, device=dev)
    row[0, 2:7] = _i32(dev, [5, 0, 3, 1, 2])
    table, n = row[:, 2:].expand(3, -1), _i32(dev, lens)
    q = torch.randn(1, Lq, H, 128, device=dev, generator=g).to(BF16).expand(3, -1, -1, -1)
    k, v = torch.randn(2, 1, Lc, H, 128, device=dev, generator=g).to(BF16).expand(2, 3, -1, -1, -1)
    mask = (torch.rand(1, 200, device=dev, generator=g) < 0.5).to(torch.uint8)
    want = _reference(q, pool, table, lens, k_cur=k, v_cur=v, cur_valid=mask)
    for m in (mask, mask.bool(), mask[:, :Lc].expand(3, -1), torch.stack([mask, mask], 2)[:, :, 0]):
        _check(ca.paged_attention(q, pool, table, n, k_cur=k, v_cur=v, cur_valid=m), want, f"{Lq} rows")
