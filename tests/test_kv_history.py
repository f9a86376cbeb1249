"""The long-history operators without a GPU: refusals, shapes of meta tensors, and
the C ABI's own argument checks."""
import ctypes

import pytest
import torch

from conftest import pkg_module

BF16 = torch.bfloat16


@pytest.fixture
def cache():
    return pkg_module("fp8_kv_cache").make_fp8_kv_block(1, 200, 2, 128, device="cpu")


def _codes(c):
    return c["k"], c["v"], c["k_scale"], c["v_scale"]


def test_bounds_refusals(cache):
    ops, hist = pkg_module("ops"), pkg_module("kv_history")
    bounds = hist.make_block_bounds(cache)
    assert bounds.shape == (1, 4, 2, 2, 128) and bounds.dtype == BF16
    assert (bounds[:, :, :, 0] == float("inf")).all() and (bounds[:, :, :, 1] == -float("inf")).all()
    with pytest.raises(ValueError, match="block"):
        hist.make_block_bounds(cache, block=96)
    for start, end in ((-1, 4), (5, 4), (0, 201)):
        with pytest.raises(ValueError, match="capacity"):
            hist.update_block_bounds(bounds, cache, start, end)
    with pytest.raises(ValueError, match="block must be"):
        hist.update_block_bounds(bounds, cache, 0, 10, block=32)
    with pytest.raises(ValueError, match="bounds must be"):
        hist.update_block_bounds(bounds[:, :3], cache, 0, 200)
    with pytest.raises(ValueError, match="bounds must be"):
        hist.update_block_bounds(bounds.float(), cache, 0, 200)
    with pytest.raises(ValueError, match="contiguous"):
        hist.update_block_bounds(bounds.transpose(3, 4).contiguous().transpose(3, 4), cache, 0, 200)
    with pytest.raises(ValueError, match="valid"):
        hist.update_block_bounds(bounds, cache, 0, 200, cache_valid=torch.ones(1, 199, dtype=torch.bool))
    with pytest.raises(TypeError, match="valid"):
        hist.update_block_bounds(bounds, cache, 0, 200, cache_valid=torch.ones(1, 200))
    with pytest.raises(ValueError, match="scales"):
        ops.kv_block_bounds_(bounds, cache["k"], cache["k_scale"][:, :9], 0, 9)
    with pytest.raises(RuntimeError, match="GPU"):
        hist.update_block_bounds(bounds, cache, 0, 200)


def test_select_refusals(cache):
    hist = pkg_module("kv_history")
    bounds = hist.make_block_bounds(cache)
    q = torch.zeros(1, 5, 4, 128, dtype=BF16)
    for kw, match in ((dict(top_k=0), "positive"), (dict(q_block=0), "positive"), (dict(keep_first=-1), "keep_first"),
                      (dict(keep_first=3, keep_last=2), "exceeds top_k"), (dict(kv_len=257), "blocks"),
                      (dict(kv_len=-1), "blocks"), (dict(block=100), "block must")):
        args = dict(kv_len=200, top_k=4)
        args.update(kw)
        with pytest.raises(ValueError, match=match):
            hist.select_blocks(q, bounds, args.pop("kv_len"), args.pop("top_k"), **args)
    with pytest.raises(TypeError, match="bf16"):
        hist.select_blocks(q.float(), bounds, 200, 4)
    with pytest.raises(ValueError, match="heads"):
        hist.select_blocks(q[:, :, :3], bounds, 200, 4)
    with pytest.raises(ValueError, match="heads"):
        hist.select_blocks(q.expand(3, -1, -1, -1), bounds.expand(2, -1, -1, -1, -1), 200, 4)
    with pytest.raises(ValueError, match="q_valid"):
        hist.select_blocks(q, bounds, 200, 4, q_valid=torch.ones(1, 4, dtype=torch.bool))
    with pytest.raises(RuntimeError, match="GPU"):
        hist.select_blocks(q, bounds, 200, 4)


def test_attention_refusals(cache):
    ca, ops = pkg_module("cache_attention"), pkg_module("ops")
    q = torch.zeros(1, 5, 4, 128, dtype=BF16)
    idx = torch.zeros(1, 2, 1, 3, dtype=torch.int32)
    kv = torch.zeros(1, 6, 2, 128, dtype=BF16)

    def call(match, exc=ValueError, q=q, cache=cache, kv_len=200, idx=idx, **kw):
        with pytest.raises(exc, match=match):
            ca.sparse_chunk_attention(q, cache, kv_len, idx, **kw)

    call("bf16 queries", TypeError, q=q.float())
    call("does not match", q=q[:, :, :3])
    call("does not match", q=q.expand(2, -1, -1, -1), cache={n: t.expand(3, -1, -1, -1) for n, t in cache.items()})
    call("capacity", kv_len=201)
    call("capacity", kv_len=-1)
    call("block must", block=48)
    call("q_block", q_block=0)
    call("block_idx", idx=idx.long())
    call("block_idx", idx=idx[:, :1])
    call("block_idx", q_block=2)
    call("softmax_scale", softmax_scale=0.0)
    call("softmax_scale", softmax_scale=float("nan"))
    call("k_cur", k_cur=kv[:, :, :1], v_cur=kv[:, :, :1])
    call("k_cur/v_cur", k_cur=kv)
    call("k_cur/v_cur", v_cur=kv)
    call("k_cur/v_cur", k_cur=kv, v_cur=kv.float())
    call("cache_valid", cache_valid=torch.ones(1, 199, dtype=torch.bool))
    call("cur_valid", k_cur=kv, v_cur=kv, cur_valid=torch.ones(1, 5, dtype=torch.bool))
    call("cache_valid", TypeError, cache_valid=torch.ones(1, 200))
    call("GPU", RuntimeError)
    with pytest.raises(TypeError, match="FP8/INT8"):
        ca.sparse_chunk_attention(q, {"k": kv, "v": kv}, 6, idx)
    with pytest.raises(ValueError, match="K and V"):
        ops.attn_kv_blocks(q, cache["k"], cache["v"][:, :100], cache["k_scale"], cache["v_scale"], 10)
    with pytest.raises(ValueError, match="K and V"):
        ops.attn_kv_blocks(q, cache["k"], cache["v"], cache["k_scale"], cache["v_scale"].double(), 10)


def test_mass_refusals(cache):
    hist = pkg_module("kv_history")
    q, lse = torch.zeros(1, 5, 4, 128, dtype=BF16), torch.zeros(1, 4, 5)

    def call(match, exc=ValueError, q=q, lse=lse, kv_len=200, **kw):
        with pytest.raises(exc, match=match):
            hist.key_mass(q, lse, cache, kv_len, **kw)

    call("expects", TypeError, q=q.float())
    call("expects", TypeError, lse=lse.double())
    call("lse", lse=lse[:, :3])
    call("does not match", q=q[:, :, :3])
    call("capacity", kv_len=201)
    call("prior", prior=torch.zeros(1, 2, 201))
    call("prior", prior=torch.zeros(1, 1, 20))
    call("prior", prior=torch.zeros(1, 2, 20, dtype=torch.float64))
    call("softmax_scale", softmax_scale=-1.0)
    call("cache_valid", cache_valid=torch.ones(1, 9, dtype=torch.bool))
    call("GPU", RuntimeError)


def test_evict_refusals(cache):
    hist, ops = pkg_module("kv_history"), pkg_module("ops")
    out = pkg_module("fp8_kv_cache").make_fp8_kv_block(1, 50, 2, 128, device="cpu")
    mass = torch.zeros(1, 2, 200)
    with pytest.raises(TypeError, match="fp32"):
        hist.evict(cache, out, mass.double(), 200, 10)
    with pytest.raises(ValueError, match="kv_len"):
        hist.evict(cache, out, mass, 201, 10)
    with pytest.raises(ValueError, match="exceeds keep"):
        hist.evict(cache, out, mass, 200, 10, keep_first=6, keep_last=5)
    with pytest.raises(ValueError, match="cache_valid"):
        hist.evict(cache, out, mass, 200, 10, cache_valid=torch.ones(2, 200, dtype=torch.bool))
    with pytest.raises(RuntimeError, match="GPU"):
        hist.evict(cache, out, mass, 200, 10)
    idx = torch.zeros(1, 2, 51, dtype=torch.int32)
    with pytest.raises(ValueError, match="capacity 50"):
        ops.move_kv_tokens_(*_codes(out), *_codes(cache), mass, idx)
    with pytest.raises(ValueError, match="idx"):
        ops.move_kv_tokens_(*_codes(out), *_codes(cache), mass, idx.long())
    with pytest.raises(ValueError, match="mass"):
        ops.move_kv_tokens_(*_codes(out), *_codes(cache), torch.zeros(1, 2, 201), idx[..., :9])
    int8 = pkg_module("fp8_kv_cache").make_int8_kv_block(1, 50, 2, 128, device="cpu")
    with pytest.raises(ValueError, match="does not match"):
        ops.move_kv_tokens_(*_codes(int8), *_codes(cache), mass, idx[..., :9])


def test_shapes_of_meta_tensors():
    ops = pkg_module("ops")

    def m(*shape, dtype=BF16):
        return torch.empty(*shape, dtype=dtype, device="meta")

    f8, f32 = torch.float8_e4m3fn, torch.float32
    c = [m(1, 200, 2, 128, dtype=f8)] * 2 + [m(1, 200, 2, 1, dtype=f32)] * 2
    q, bounds = m(3, 70, 4, 128), m(1, 4, 2, 2, 128)
    ops.kv_block_bounds_(bounds, c[0], c[2], 0, 200)
    idx = ops.select_kv_blocks(q, bounds, 200, 3, 64, 32)
    assert idx.shape == (3, 2, 3, 3) and idx.dtype == torch.int32
    out, lse = ops.attn_kv_blocks(q, *c, 200, idx, 64, 32)
    assert out.shape == q.shape and lse.shape == (3, 4, 70) and lse.dtype == f32
    mass = ops.attn_key_mass(q, lse, c[0], c[2], 200)
    assert mass.shape == (1, 2, 200)
    kept = ops.select_kv_tokens(mass, 200, 50)
    assert kept.shape == (1, 2, 50) and kept.dtype == torch.int32
    assert ops.move_kv_tokens_(*c, *c, mass, kept).shape == (1, 2, 50)


_A = 0x10000  # a fake device address: every call below is refused before it is touched


def test_c_abi_refusals():
    lib = pkg_module("_lib").load()

    def err():
        return lib.hn_last_error().decode()

    st = (ctypes.c_int64 * 4)(256, 256, 128, 1)
    s3 = (ctypes.c_int64 * 3)(2, 2, 1)
    bs = (ctypes.c_int64 * 5)(512, 512, 256, 128, 1)

    def bounds(fmt=0, D=128, cap=100, start=0, end=100, block=64, n=2, vs=0, cs=st, kc=_A):
        return lib.hn_kv_block_bounds(fmt, kc, cs, _A, s3, 1, 2, D, cap, start, end, block, None, vs, _A, bs, n, None)

    for kw, match in ((dict(fmt=5), "format"), (dict(D=64), "head dim"), (dict(block=63), "block"),
                      (dict(block=2048), "block"), (dict(end=101), "capacity"), (dict(start=-1), "shape"),
                      (dict(start=101, end=100), "shape"), (dict(n=1), "few blocks"), (dict(vs=-1), "stride"),
                      (dict(kc=_A + 1), "misaligned"), (dict(cs=(ctypes.c_int64 * 4)(256, 250, 128, 1)), "multiples")):
        assert bounds(**kw) == -1 and match in err(), kw
    assert bounds(start=100, end=100, kc=None) == 0

    def select(D=128, Hq=4, H=2, blocks=9, q_block=1, k=4, first=0, last=0, ws=_A, wsb=1 << 20, q=_A):
        return lib.hn_select_kv_blocks(q, st, 1, 3, Hq, D, None, 0, _A, bs, H, blocks, q_block, k, first, last, _A, ws,
                                       wsb, None)

    for kw, match in ((dict(D=96), "head dim"), (dict(Hq=3), "shape"), (dict(q_block=0), "positive"),
                      (dict(k=0), "positive"), (dict(k=(1 << 31) - 1), "too many"), (dict(blocks=1 << 30), "too many"),
                      (dict(first=3, last=2), "exceeds"), (dict(last=-1), "exceeds"),
                      (dict(wsb=64), "workspace"), (dict(ws=_A + 8), "workspace"), (dict(q=None), "null")):
        assert select(**kw) == -1 and match in err(), kw
    assert lib.hn_select_kv_blocks_workspace_size(1, 2, 3, 9) >= 6 * (2048 + 36)
    assert lib.hn_select_kv_blocks_workspace_size(1, 2, 3, 0) == 0

    def attn(D=128, Hq=4, H=2, cap=100, kv=100, block=64, q_block=8, k=3, scale=0.1, cvs=0, q=_A, lse=_A, cs=st):
        return lib.hn_attn_kv_blocks(0, q, st, 1, 3, Hq, D, _A, _A, cs, _A, _A, s3, H, cap, kv, None, cvs, _A, s3, k,
                                     block, q_block, None, None, None, 0, None, 0, scale, _A, st, lse, None, 0, None)

    for kw, match in ((dict(D=64), "head dim"), (dict(Hq=5), "shape"), (dict(kv=101), "capacity"),
                      (dict(block=65), "block"), (dict(q_block=0), "q_block"), (dict(k=-2), "too many"),
                      (dict(scale=0.0), "softmax_scale"), (dict(scale=float("inf")), "softmax_scale"),
                      (dict(cvs=-1), "stride"), (dict(q=_A + 8), "misaligned"), (dict(lse=None), "null"),
                      (dict(cs=(ctypes.c_int64 * 4)(256, 0, 128, 1)), "strides")):
        assert attn(**kw) == -1 and match in err(), kw
    assert lib.hn_attn_kv_blocks_workspace_size(1, 1, 4, 3, 100, 0, 3, 64, 1) == 0   # heads do not divide

    def mass(D=128, Bq=2, B=1, Hq=4, kv=100, prior_len=0, prior=None, scale=0.1, lse=_A):
        return lib.hn_attn_key_mass(0, _A, st, Bq, 3, Hq, D, lse, _A, st, _A, s3, B, 2, 100, kv, None, 0, scale, prior,
                                    s3 if prior_len else None, prior_len, _A, None, 0, None)

    for kw, match in ((dict(D=64), "head dim"), (dict(Bq=3, B=2), "divide"), (dict(kv=101), "capacity"),
                      (dict(prior_len=101), "prior"), (dict(prior_len=5), "null"), (dict(scale=-1.0), "softmax_scale"),
                      (dict(lse=None), "null"), (dict(Hq=3), "shape")):
        assert mass(**kw) == -1 and match in err(), kw
    assert mass(kv=0, lse=None) == 0

    def tokens(kv=100, keep=10, first=0, last=0, m=_A):
        return lib.hn_select_kv_tokens(m, s3, 1, 2, kv, None, 0, keep, first, last, _A, None, 0, None)

    for kw, match in ((dict(kv=-1), "shape"), (dict(first=6, last=5), "exceeds"), (dict(m=None), "null"),
                      (dict(m=_A + 2), "misaligned"), (dict(kv=1 << 20), "workspace")):
        assert tokens(**kw) == -1 and match in err(), kw
    assert tokens(keep=0, m=None) == 0

    far = _A << 12

    def move(D=128, keep=10, cap=10, os=st, k=_A, out=far, out_scale=far):
        return lib.hn_move_kv_tokens(k, _A, st, _A, _A, s3, _A, s3, 1, 2, D, 100, _A, keep, out, far, os, out_scale,
                                     far, s3, cap, far, None)

    for kw, match in ((dict(D=64), "head dim"), (dict(keep=11), "capacity"), (dict(k=None), "null"),
                      (dict(os=(ctypes.c_int64 * 4)(256, 248, 128, 1)), "multiples"),
                      # 100 tokens of 256 bytes and 800 of scales from _A on
                      (dict(out=_A + 99 * 256), "overlaps"), (dict(out=_A - 10 * 256 + 16), "overlaps"),
                      (dict(out_scale=_A + 796), "overlaps")):
        assert move(**kw) == -1 and match in err(), kw
    assert move(keep=0, k=None) == 0


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the refusal on a machine without a GPU")
def test_no_gfx950_device_is_refused():
    L = pkg_module("_lib")
    lib = L.load()
    st = (ctypes.c_int64 * 4)(256, 256, 128, 1)
    s3 = (ctypes.c_int64 * 3)(2, 2, 1)
    assert lib.hn_select_kv_tokens(_A, s3, 1, 2, 100, None, 0, 10, 0, 0, _A, None, 0, None) == L.HN_E_DEVICE
    assert lib.hn_kv_block_bounds(0, _A, st, _A, s3, 1, 2, 128, 100, 0, 100, 64, None, 0, _A,
                                  (ctypes.c_int64 * 5)(512, 512, 256, 128, 1), 2, None) == L.HN_E_DEVICE


def test_model_refusals():
    dit, hist = pkg_module("dit_block"), pkg_module("kv_history")
    kvc = pkg_module("fp8_kv_cache")
    cache = kvc.make_fp8_kv_block(1, 256, 2, 128, device="cpu")
    with pytest.raises(ValueError, match="exceeds top_k"):
        hist.LayerHistory(cache, top_k=2, keep_first=1, keep_last=2)
    h = hist.LayerHistory(cache, top_k=4)
    with pytest.raises(ValueError, match="mass"):
        h.evict(cache, cache, 128, 64)
    for kw in (dict(top_k=-1), dict(keep_first=-1), dict(keep_last=-1), dict(q_block=0)):
        with pytest.raises(ValueError, match="must"):
            hist.LayerHistory(cache, **{"top_k": 4, **kw})
    # passes over tokens that bounds and mass do not account for
    h = hist.LayerHistory(cache, top_k=4, track_mass=True)
    q = torch.zeros(1, 3, 2, 128, dtype=torch.bfloat16)
    for update in (False, True):
        with pytest.raises(ValueError, match="accounts for 0 tokens, the pass reads 64"):
            h.attend(q, q, q, cache, 64, update)
    h.mass, h.length = torch.ones(1, 2, 128), 128        # as after a roll-out
    with pytest.raises(ValueError, match="accounts for 128 tokens, not 100"):
        h.evict(cache, cache, 100, 64)
    with pytest.raises(RuntimeError, match="GPU"):       # (a new roll-out: allowed, and on a GPU it would run)
        h.attend(q, q, q, cache, 0, True)
    assert h.mass is None and h.length == 0
    h.reset(cache, 0)
    assert h.length == 0 and h.mass is None
    block = dit.FP8DiTBlock.__new__(dit.FP8DiTBlock)
    with pytest.raises(ValueError, match="image-only"):
        dit.FP8DiTBlock.forward(block, None, None, None, None, cache, 0, txt=1, history=h)


def test_model_looks_at_every_layer_before_it_cuts_one():
    """(with caches on the CPU, the first move would be refused there)"""
    dit, hist = pkg_module("dit_block"), pkg_module("kv_history")
    kvc = pkg_module("fp8_kv_cache")
    m = dit.FP8ARModel.__new__(dit.FP8ARModel)
    m.evict_keep, m.latent_shape, m.write_tokens, m.cache_valid_len = 32, (1, 4, 8), 32, 64
    m.caches = [kvc.make_fp8_kv_block(1, 96, 2, 128, device="cpu") for _ in range(3)]
    m.spare = kvc.make_fp8_kv_block(1, 96, 2, 128, device="cpu")
    m.histories = [hist.LayerHistory(c, track_mass=True) for c in m.caches]
    for h in m.histories:
        h.mass, h.length = torch.ones(1, 2, 64), 64
    m.histories[2].length = 60
    with pytest.raises(ValueError, match="accounts for 60 tokens, not 64"):
        m.evict_history()
    m.histories[2].length, m.histories[1].mass = 64, None
    with pytest.raises(ValueError, match="needs the mass"):
        m.evict_history()
    m.histories[1].mass = torch.ones(1, 2, 64)
    with pytest.raises(RuntimeError, match="GPU"):
        m.evict_history()


def test_model_looks_at_the_schedule_before_it_cuts():
    dit = pkg_module("dit_block")
    m = dit.FP8ARModel.__new__(dit.FP8ARModel)
    m.cache_valid_len, m.tokens_per_chunk, m.write_tokens, m.capacity, m.evict_keep = 20, 10, 10, 25, 8
    m.heads, m.head_dim = 2, 128
    cut = []
    m.evict_history = lambda: cut.append(1)
    noise = torch.zeros(1, 10, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="sigmas"):
        m.generate_chunk(noise, [None], None, [1.0])
    for bad in (noise[:, :9], noise[..., :128], noise[0], noise.expand(2, -1, -1)):
        with pytest.raises(ValueError, match="noise"):
            m.generate_chunk(bad, [], None, [1.0])
    assert not cut
    with pytest.raises(ValueError, match="capacity"):     # (this stub makes no room)
        m.generate_chunk(noise, [], None, [1.0])
    assert cut == [1]


def test_layer_history_commit_counts_all_of_a_pass_or_nothing():
    """A commit whose bounds cannot be brought up to date (here: of a cache that is not on
    the GPU) leaves the history as it was, and can be called again."""
    hist, kvc = pkg_module("kv_history"), pkg_module("fp8_kv_cache")
    cache = kvc.make_fp8_kv_block(1, 256, 2, 128, device="cpu")
    h = hist.LayerHistory(cache, top_k=4, track_mass=True)
    old, new = torch.ones(1, 2, 64), torch.ones(1, 2, 96)
    h.mass, h.length, h._written = old, 64, (new, 64, 96)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="GPU"):
            h.commit(cache)
        assert h.mass is old and h.length == 64 and h._written[0] is new
    h.rollback()
    h.commit(cache)
    assert h.mass is old and h.length == 64


def test_layer_history_mass_is_fp32_whatever_the_default():
    hist, kvc = pkg_module("kv_history"), pkg_module("fp8_kv_cache")
    h = hist.LayerHistory(kvc.make_fp8_kv_block(1, 64, 2, 128, device="cpu"), track_mass=True)
    for dtype in (torch.bfloat16, torch.float64):
        torch.set_default_dtype(dtype)
        try:
            h.reset(kvc.make_fp8_kv_block(1, 64, 2, 128, device="cpu"), 10)
        finally:
            torch.set_default_dtype(torch.float32)
        assert h.mass.dtype == torch.float32 and h.mass.shape == (1, 2, 10)
