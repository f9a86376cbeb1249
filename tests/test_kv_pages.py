"""The paged cache without a GPU: refusals, shapes of meta tensors, the C ABI's argument
checks, and the host's bookkeeping of pages against a plain model of it."""
import ctypes
import random

import pytest
import torch

from conftest import pkg_module

BF16, I32 = torch.bfloat16, torch.int32


@pytest.fixture
def pool():
    return pkg_module("kv_pages").make_pages(6, 2, page=64, device="cpu")


def _codes(c):
    return c["k"], c["v"], c["k_scale"], c["v_scale"]


def test_pools():
    kp = pkg_module("kv_pages")
    pool = kp.make_pages(6, 3, page=128, layers=2, device="cpu")
    assert pool["k"].shape == (2, 6, 128, 3, 128) and pool["k"].dtype == torch.float8_e4m3fn
    assert pool["v_scale"].shape == (2, 6, 128, 3, 1) and pool["v_scale"].stride(2) == 1
    assert kp.make_pages(1, 1, code_dtype=torch.int8, device="cpu")["v"].dtype == torch.int8
    with pytest.raises(ValueError, match="page must"):
        kp.make_pages(6, 3, page=96, device="cpu")
    with pytest.raises(TypeError, match="int8"):
        kp.make_pages(6, 3, code_dtype=BF16, device="cpu")


def test_write_refusals(pool):
    kp, ops = pkg_module("kv_pages"), pkg_module("ops")
    kv = torch.zeros(3, 5, 2, 128, dtype=BF16)
    table, start = torch.zeros(3, 2, dtype=I32), torch.zeros(3, dtype=I32)

    def call(match, exc=ValueError, pool=pool, k=kv, v=kv, table=table, start=start, **kw):
        with pytest.raises(exc, match=match):
            kp.write_pages(pool, k, v, table, start, **kw)

    call("bf16", TypeError, k=kv.float())
    call("k and v", k=kv[:, :, :1], v=kv[:, :, :1])
    call("k and v", v=kv[:, :4])
    call("k and v", k=kv[0], v=kv[0])
    call("table", table=table.long())
    call("table", table=table[:2])
    call("table", table=table[0])
    call("start", start=start.long())
    call("start", start=start[:2])
    call("counts", counts=start.float())
    call("status", TypeError, status=torch.zeros(1))
    call("codes must be", TypeError, pool={n: t.float() for n, t in pool.items()})
    call("page must", pool=kp.make_pages(6, 2, page=64, device="cpu") | {n: t[:, :48] for n, t in pool.items()})
    call("K and V", pool=pool | {"v": pool["v"][:5]})
    call("scales", pool=pool | {"k_scale": pool["k_scale"].double()})
    call("GPU", RuntimeError)
    with pytest.raises(ValueError, match="scales"):
        ops.kv_pages_write_(pool["k"][0], pool["v"][0], pool["k_scale"], pool["v_scale"], kv, kv, table, start)


def test_attention_refusals(pool):
    ca = pkg_module("cache_attention")
    q = torch.zeros(3, 5, 4, 128, dtype=BF16)
    table, n = torch.zeros(3, 2, dtype=I32), torch.zeros(3, dtype=I32)
    kv = torch.zeros(3, 6, 2, 128, dtype=BF16)

    def call(match, exc=ValueError, q=q, pool=pool, table=table, n=n, **kw):
        with pytest.raises(exc, match=match):
            ca.paged_attention(q, pool, table, n, **kw)

    call("bf16 queries", TypeError, q=q.float())
    call("must be", q=q[0])
    call("does not match", q=q[:, :, :3])
    call("does not match", q=q[..., :64])
    call("table", table=table[:2])
    call("table", table=table.long())
    call("kv_len", n=n[:2])
    call("kv_len", n=n.long())
    call("softmax_scale", softmax_scale=0.0)
    call("softmax_scale", softmax_scale=float("inf"))
    call("k_cur", k_cur=kv[:, :, :1], v_cur=kv[:, :, :1])
    call("k_cur", k_cur=kv[:2], v_cur=kv[:2])
    call("k_cur/v_cur", k_cur=kv)
    call("k_cur/v_cur", v_cur=kv)
    call("k_cur/v_cur", k_cur=kv, v_cur=kv.float())
    call("no tail", causal=True, k_cur=kv, v_cur=kv)
    call("cur_valid", k_cur=kv, v_cur=kv, cur_valid=torch.ones(3, 5, dtype=torch.bool))
    call("cur_valid", TypeError, k_cur=kv, v_cur=kv, cur_valid=torch.ones(3, 6))
    call("GPU", RuntimeError)
    call("FP8/INT8", TypeError, pool={"k": kv, "v": kv})


def test_copy_and_read_refusals(pool):
    kp = pkg_module("kv_pages")

    def call(match, src, dst, pool=pool, exc=ValueError):
        with pytest.raises(exc, match=match):
            kp.copy_pages(pool, src, dst)

    call("one length", [0, 1], [2])
    call("lie in", [0], [6])
    call("lie in", [-1], [2])
    call("twice", [0, 1], [2, 2])
    call("twice", [0, 1], [1, 2])
    call("twice", [3], [3])
    call("scales", [0], [1], pool | {"k_scale": pool["k_scale"][:5]})
    call("K and V", [0], [1], pool | {"v": pool["v"].view(torch.int8)})
    call("GPU", [0], [1], exc=RuntimeError)
    kp.copy_pages(pool, [], [])
    n = torch.zeros(3, dtype=I32)
    with pytest.raises(ValueError, match="Invalid KV key"):
        kp.read_pages(pool, "q", torch.zeros(3, 2, dtype=I32), n, 5)
    with pytest.raises(ValueError, match="max_len"):
        kp.read_pages(pool, "k", torch.zeros(3, 2, dtype=I32), n, -1)
    with pytest.raises(ValueError, match="kv_len"):
        kp.read_pages(pool, "k", torch.zeros(2, 2, dtype=I32), n, 5)
    with pytest.raises(ValueError, match="table"):
        kp.read_pages(pool, "k", torch.zeros(3, 2), n, 5)
    with pytest.raises(RuntimeError, match="GPU"):
        kp.read_pages(pool, "k", torch.zeros(3, 2, dtype=I32), n, 5)


def test_a_page_is_one_run_of_memory():
    ops = pkg_module("ops")
    t = torch.empty(3, 7, 64, 5, 128, dtype=torch.uint8)
    assert ops._page_bytes(t, "x") == (7 * 64 * 5 * 128, 64 * 5 * 128, 64 * 5 * 128)
    s = torch.empty(3, 7, 5, 64, 1).transpose(2, 3)
    assert ops._page_bytes(s, "x") == (7 * 64 * 5 * 4, 64 * 5 * 4, 64 * 5 * 4)
    assert ops._page_bytes(t[:1, :1], "x")[2] == 64 * 5 * 128
    assert ops._page_bytes(t[:, ::2], "x") == (7 * 64 * 5 * 128, 2 * 64 * 5 * 128, 64 * 5 * 128)
    with pytest.raises(ValueError, match="run of memory"):
        ops._page_bytes(t[:, :, :, :3], "x")


def test_shapes_of_meta_tensors():
    ops = pkg_module("ops")
    meta = dict(device="meta")
    codes = torch.empty(6, 64, 2, 128, dtype=torch.int8, **meta)
    scale = torch.empty(6, 64, 2, 1, **meta)
    table, n = torch.empty(3, 2, dtype=I32, **meta), torch.empty(3, dtype=I32, **meta)
    q = torch.empty(3, 5, 4, 128, dtype=BF16, **meta)
    out, lse = ops.attn_kv_pages(q, codes, codes, scale, scale, table, n)
    assert out.shape == q.shape and lse.shape == (3, 4, 5) and lse.dtype == torch.float32
    y = ops.kv_pages_read(codes, scale, table, n, 70)
    assert y.shape == (3, 70, 2, 128) and y.dtype == BF16
    kv = torch.empty(3, 5, 2, 128, dtype=BF16, **meta)
    assert ops.kv_pages_write_(codes, codes.clone(), scale, scale.clone(), kv, kv, table, n) is None
    assert ops.kv_pages_copy_(codes, codes.clone(), scale, scale.clone(), [0], [1]) is None


def test_c_abi_checks():
    L = pkg_module("_lib")
    lib = L.load()
    P = ctypes.c_void_p(256)
    st = (ctypes.c_int64 * 4)(16384, 256, 128, 1)
    odd = (ctypes.c_int64 * 4)(16384, 248, 120, 1)

    def err():
        return lib.hn_last_error().decode()

    def write(fmt=0, D=128, H=2, B=1, xs=st, cs=st, page=64, width=2, k=P, start=P, mode=1, n=5,
              status=None, ws=None, nbytes=0):
        return lib.hn_kv_pages_write(fmt, k, P, xs, B, n, H, D, P, P, cs, P, P, st, 6, page, P, 2, width, start, None,
                                     mode, status, ws, nbytes, None)

    for kw, match in ((dict(fmt=3), "format"), (dict(D=64), "head dim"), (dict(H=0), "shape"), (dict(page=32), "page"),
                      (dict(page=96), "page"), (dict(width=-1), "table"), (dict(width=2 ** 31), "table"),
                      (dict(cs=odd), "multiples of 16"), (dict(xs=(ctypes.c_int64 * 4)(9, 9, 9, 1)), "multiples of 8"),
                      (dict(k=ctypes.c_void_p(8)), "misaligned"), (dict(start=None), "null"), (dict(mode=0), "scale mode")):
        assert write(**kw) == L.HN_E_ARG and match in err(), kw
    assert write(B=0) == 0
    size = lib.hn_kv_pages_write_workspace_size
    assert size(1, 256, 2) == 0 and size(1, 257, 2) == 16 and size(1, 65, 8) == 16 and size(2, 65, 9) == 48 and size(1, 2 ** 20, 2) == 0 and size(0, 9, 9) == 0
    for kw in (dict(ws=None, nbytes=16), dict(ws=P, nbytes=15), dict(ws=ctypes.c_void_p(8), nbytes=16)):
        assert write(n=257, status=P, **kw) == L.HN_E_ARG and "workspace" in err(), kw

    def attend(page=64, D=128, Hq=4, causal=0, cur=0, scale=0.1, q=P, cs=st, ws=None, nbytes=0, width=2, Lq=1,
               first=None):
        return lib.hn_attn_kv_pages(0, q, st, 1, Lq, Hq, D, P, P, cs, P, P, st, 2, 6, page, P, 2, width, P, causal, first,
                                    P if cur else None, P if cur else None, st if cur else None, cur, None, 0, scale, P,
                                    st, P, ws, nbytes, None)

    for kw, match in ((dict(page=48), "page"), (dict(D=96), "head dim"), (dict(Hq=3), "shape"),
                      (dict(causal=1, cur=3), "no tail"), (dict(first=P), "q_start"),
                      (dict(causal=1, first=ctypes.c_void_p(2)), "misaligned"), (dict(scale=0.0), "softmax_scale"),
                      (dict(scale=float("nan")), "softmax_scale"), (dict(q=ctypes.c_void_p(8)), "misaligned"),
                      (dict(cs=odd), "multiples of 16"), (dict(width=2 ** 28), "too many keys"), (dict(q=None), "null"),
                      (dict(width=300), "workspace")):
        assert attend(**kw) == L.HN_E_ARG and match in err(), kw
    assert lib.hn_attn_kv_pages_workspace_size(1, 1, 4, 2, 128, 0) == 0
    assert lib.hn_attn_kv_pages_workspace_size(1, 1, 4, 2, 1 << 16, 0) > 0
    assert lib.hn_attn_kv_pages_workspace_size(0, 1, 4, 2, 128, 0) == 0

    four = ctypes.c_void_p * 4
    sizes = (ctypes.c_int64 * 4)(16384, 16384, 512, 512)
    one = (ctypes.c_int32 * 1)

    def copy(base=four(256, 256, 256, 256), page=sizes, size=sizes, src=0, dst=1, layers=1):
        return lib.hn_kv_pages_copy(base, sizes, page, size, layers, 6, one(src), one(dst), 1, None)

    for kw, match in ((dict(base=four(256, 8, 256, 256)), "multiples of 16"), (dict(src=6), "outside"),
                      (dict(dst=-1), "outside"), (dict(page=(ctypes.c_int64 * 4)(8192, 16384, 512, 512)), "overlap"),
                      (dict(layers=70000), "layers"), (dict(layers=-1), "shape")):
        assert copy(**kw) == L.HN_E_ARG and match in err(), kw
    assert copy(layers=0) == 0
    assert lib.hn_kv_pages_read(0, P, st, P, st, 6, 64, P, 2, 2, P, 1, -1, 2, 128, P, None) == L.HN_E_ARG
    assert lib.hn_kv_pages_read(0, P, st, P, st, 6, 64, P, 2, 2, P, 1, 0, 2, 128, P, None) == 0


# --------------------------------------------------------------------------
# the host's bookkeeping

class Tokens:
    """What every place of a pool holds, as numbers: writes through a batch's table."""

    def __init__(self, monkeypatch, cache):
        self.cache, self.at, self.copies = cache, {}, 0
        monkeypatch.setattr(pkg_module("kv_pages"), "copy_pages", self.copy)

    def copy(self, pool, src, dst):
        assert len(set(dst)) == len(dst) and not set(dst) & set(src)
        self.copies += len(src)
        new = {(d, i): self.at.get((s, i)) for s, d in zip(src, dst) for i in range(self.cache.page)}
        self.at.update(new)

    def write(self, batch, values):
        for row, start, vals in zip(batch.table.tolist(), batch.start.tolist(), values):
            for j, v in enumerate(vals):
                page = row[(start + j) // self.cache.page]
                assert page >= 0
                self.at[page, (start + j) % self.cache.page] = v

    def read(self, batch):
        return [[self.at[row[t // self.cache.page], t % self.cache.page] for t in range(n)]
                for row, n in zip(batch.table.tolist(), batch.start.tolist())]


def _whole(cache):
    """Every page is free or held as often as it is counted."""
    held = [p for t in cache._table.values() for p in t]
    assert [held.count(p) for p in range(cache.pages)] == cache._refs
    assert sorted(cache._free) == [p for p in range(cache.pages) if not cache._refs[p]]


@pytest.mark.parametrize("seed", range(8))
def test_sequences_keep_their_tokens(monkeypatch, seed):
    """Random runs of appends, forks, cuts, frees, abandoned passes and compactions: every
    sequence reads what was appended to it, whatever others do with shared pages."""
    kp = pkg_module("kv_pages")
    rng = random.Random(seed)
    cache = kp.PagedKVCache(2, 40, 1, page=64, device="cpu")
    tokens, want, stamp = Tokens(monkeypatch, cache), {}, iter(range(10 ** 9))
    for _ in range(300):
        act = rng.choice(["new", "append", "append", "append", "append", "fork", "cut", "free", "discard", "compact"])
        seqs = list(want)
        if act == "new" and len(seqs) < 8:
            want[cache.new()] = []
        elif act == "fork" and seqs and len(seqs) < 8:
            s = rng.choice(seqs)
            want[cache.fork(s)] = list(want[s])
        elif act == "cut" and seqs:
            s = rng.choice(seqs)
            n = rng.randrange(len(want[s]) + 1)
            cache.truncate(s, n)
            del want[s][n:]
        elif act == "free" and len(seqs) > 2:
            s = rng.choice(seqs)
            cache.free(s)
            del want[s]
        elif act == "compact":
            cache.compact()
            used = [p for p in range(cache.pages) if cache._refs[p]]
            assert used == list(range(len(used)))
        elif act in ("append", "discard") and seqs:
            some = rng.sample(seqs, rng.randrange(1, len(seqs) + 1))
            adds = [rng.choice([0, 1, 5, 63, 64, 130]) for _ in some]
            if rng.random() < 0.3:
                adds = [rng.choice([1, 70])] * len(some)
            before = {s: list(t) for s, t in cache._table.items()}, list(cache._refs), cache.free_pages
            try:
                batch = cache.open(some, adds)
            except ValueError as e:
                assert "pages are needed" in str(e)
                assert before == ({s: list(t) for s, t in cache._table.items()}, list(cache._refs), cache.free_pages)
                continue
            assert (batch.counts is None) == (len(set(adds)) <= 1)
            vals = [[next(stamp) for _ in range(a)] for a in adds]
            tokens.write(batch, vals)
            if act == "append":
                batch.commit()
                for s, v in zip(some, vals):
                    want[s] += v
            else:
                batch.discard()
            with pytest.raises(ValueError, match="past"):
                batch.commit()
        _whole(cache)
        if want:
            assert [cache.length(s) for s in want] == [len(v) for v in want.values()]
            assert tokens.read(cache.open(list(want))) == list(want.values())
    assert tokens.copies > 0


def test_forks_share_until_they_write(monkeypatch):
    kp = pkg_module("kv_pages")
    cache = kp.PagedKVCache(1, 10, 1, page=64, device="cpu")
    tokens = Tokens(monkeypatch, cache)
    a = cache.new()
    batch = cache.open([a], 100)
    tokens.write(batch, [list(range(100))])
    batch.commit()
    b, c = cache.fork(a), cache.fork(a)
    assert cache.free_pages == 8 and tokens.copies == 0
    batch = cache.open([a, b, c], 1)  # the half page: two copies, the last holder keeps it
    assert tokens.copies == 2 and cache.free_pages == 6
    batch.commit()
    cache.open([a, b, c], 1).commit()
    assert tokens.copies == 2
    cache.free(a)
    cache.free(b)
    assert cache.free_pages == 8
    full = cache.new()
    cache.open([full], 64 * 8).commit()
    with pytest.raises(ValueError, match="1 pages are needed, 0 are free"):
        cache.open([full], 1)
    d = cache.fork(full)  # a whole last page is not copied by the next token
    cache.free(c)
    copies = tokens.copies
    cache.open([d], 1).commit()
    assert tokens.copies == copies and cache.length(full) == 512 and cache.length(d) == 513


def test_cache_refusals():
    kp = pkg_module("kv_pages")
    with pytest.raises(ValueError, match="positive"):
        kp.PagedKVCache(0, 4, 1, device="cpu")
    cache = kp.PagedKVCache(1, 4, 1, device="cpu")
    a, b = cache.new(), cache.new()
    for call in (lambda: cache.open([7]), lambda: cache.fork(7), lambda: cache.free(7), lambda: cache.truncate(7, 0),
                 lambda: cache.length(7)):
        with pytest.raises(ValueError, match="no sequence"):
            call()
    with pytest.raises(ValueError, match="tokens"):
        cache.open([a, b], [1])
    with pytest.raises(ValueError, match="tokens"):
        cache.open([a], -1)
    with pytest.raises(ValueError, match="once"):
        cache.open([a, a], 1)
    assert cache.open([a, a]).table.shape == (2, 0)
    with pytest.raises(ValueError, match="cannot keep"):
        cache.truncate(a, 1)
    batch = cache.open([a, b], [3, 5])
    kv = torch.zeros(2, 4, 1, 128, dtype=BF16)
    with pytest.raises(ValueError, match="opened for"):
        batch.write(0, kv, kv)
    same = cache.open([a, b], 3)
    with pytest.raises(ValueError, match="opened for"):
        same.write(0, kv, kv)
    same.commit()
    with pytest.raises(ValueError, match="past"):
        batch.write(0, torch.zeros(2, 5, 1, 128, dtype=BF16), torch.zeros(2, 5, 1, 128, dtype=BF16))
    cache.free(a)
    with pytest.raises(ValueError, match="past"):
        same.attend(0, torch.zeros(2, 1, 1, 128, dtype=BF16))


def test_a_sequence_grows_in_one_pass_at_a_time():
    """A second pass would write the same places: the first is refused from then on, passes
    that only read are not, and what the refused one took is the sequence's room."""
    kp = pkg_module("kv_pages")
    cache = kp.PagedKVCache(1, 6, 1, device="cpu")
    a, b = cache.new(), cache.new()
    cache.open([a, b], [70, 3]).commit()
    reader, first = cache.open([a, b]), cache.open([a, b], [100, 0])
    second = cache.open([a], 2)
    for call in (first.commit, first.discard, lambda: first.attend(0, torch.zeros(2, 1, 1, 128, dtype=BF16))):
        with pytest.raises(ValueError, match="grow again"):
            call()
    other = cache.open([b], 1)  # (first adds nothing to b)
    reader._check()
    second.commit()
    other.commit()
    assert cache.length(a) == 72 and cache.length(b) == 4
    with pytest.raises(ValueError, match="past"):
        reader._check()
    cache.truncate(a, 72)
    assert cache.free_pages == 6 - 2 - 1
    with pytest.raises(ValueError, match="needed"):
        cache.open([a], 64 * 5)
    last = cache.open([a], 1)  # (a pass that is refused for want of room leaves others valid)
    with pytest.raises(ValueError, match="needed"):
        cache.open([a], 64 * 5)
    last.commit()
    assert cache.length(a) == 73


def test_model_refusals():
    db = pkg_module("dit_block")
    for kw in (dict(text_len=4), dict(sparse_top_k=2), dict(evict_keep=2)):
        with pytest.raises(ValueError, match="pages apply"):
            db.FP8ARModel(0, 256, 2, (1, 2, 2), 2, pages=4, device="cpu", **kw)
    plain = db.FP8ARModel(0, 256, 2, (1, 2, 2), 2, device="cpu")
    for call in (plain.start_branch, lambda: plain.fork_branch(0), lambda: plain.drop_branch(0)):
        with pytest.raises(ValueError, match="branches need"):
            call()
    with pytest.raises(ValueError, match="steps branches"):
        plain.generate_chunk(torch.zeros(1, 4, 256), [], None, [0.0], branches=[0])


@pytest.mark.parametrize("adds,rows,at_start", [([7, 5], 7, True), ([7, 5], 16, True), ([7, 0], 8, True),
                                                ([7, 5], 6, False), ([7, 7], 7, False), ([7, 7], 16, False),
                                                ([0, 0], 3, False)])
def test_where_causal_queries_of_a_batch_stand(monkeypatch, adds, rows, at_start):
    """Sequences that add different numbers of tokens: as many queries as the longest adds,
    or more of them (padding), start at each sequence's first new token, as write's rows do."""
    kp, ca = pkg_module("kv_pages"), pkg_module("cache_attention")
    cache = kp.PagedKVCache(1, 8, 1, page=64, device="cpu")
    seqs = [cache.new(), cache.new()]
    cache.open(seqs, [20, 3]).commit()
    batch, seen = cache.open(seqs, adds), []
    monkeypatch.setattr(kp, "write_pages", lambda *a, **kw: None)
    monkeypatch.setattr(ca, "paged_attention", lambda *a, **kw: seen.append((a[3].tolist(), kw["q_start"])))
    kv = torch.zeros(2, max(max(adds), rows if len(set(adds)) > 1 else 0), 1, 128, dtype=BF16)
    batch.write(0, kv, kv)
    batch.attend(0, torch.zeros(2, rows, 1, 128, dtype=BF16), causal=True)
    (end, start), = seen
    assert end == [20 + adds[0], 3 + adds[1]]
    assert (start.tolist() == [20, 3]) if at_start else start is None


def test_a_pass_ends_no_pass_of_a_sequence_that_it_only_reads():
    """commit and discard leave sequences alone to which their batch adds nothing: the room
    that another pass took for one, and that pass, stand."""
    kp = pkg_module("kv_pages")
    for end in ("commit", "discard"):
        cache = kp.PagedKVCache(1, 12, 1, device="cpu")
        a, b = cache.new(), cache.new()
        cache.open([a, b], [70, 3]).commit()
        grows, reads, twice, mixed = cache.open([b], 200), cache.open([b]), cache.open([a, a]), cache.open([a, b], [9, 0])
        room, free = list(cache._table[b]), cache.free_pages
        for batch in (reads, twice, mixed):
            getattr(batch, end)()
            assert cache._table[b] == room and cache.free_pages == free
            with pytest.raises(ValueError, match="past"):  # (it is over itself)
                getattr(batch, end)()
        assert cache.length(a) == (79 if end == "commit" else 70) and cache.length(b) == 3
        grows.commit()
        assert cache.length(b) == 203
        _whole(cache)


def test_a_cache_is_on_its_pools_device():
    """Whatever the name that it was given ("cuda" is another device once the current one
    changes): the tables of later passes go where the pages are."""
    cache = pkg_module("kv_pages").PagedKVCache(1, 4, 1, device="cpu:0")
    assert cache.device == cache.pool["k"].device == cache.open([cache.new()], 3).table.device


def test_no_pass_is_captured(monkeypatch):
    """A replay would bring the tables of the recorded pass again, from host memory that is
    another's by then, and repeat its copies: refused, with nothing changed."""
    cache = pkg_module("kv_pages").PagedKVCache(1, 6, 1, device="cpu")
    a = cache.new()
    cache.open([a], 70).commit()
    b = cache.fork(a)
    state = list(cache._refs), {s: list(t) for s, t in cache._table.items()}, list(cache._free)
    monkeypatch.setattr(cache, "device", torch.device("cuda", 0))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for call in (lambda: cache.open([b], 1), lambda: cache.open([b]), cache.compact):
        with pytest.raises(RuntimeError, match="captured"):
            call()
    assert state == (cache._refs, cache._table, cache._free)
