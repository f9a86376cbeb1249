"""Long-history operators of the quantized KV cache, as a program calls them.

A roll-out outlives any fixed cache: its denoising passes read a few blocks of
the history instead of all of it, and a full cache keeps the tokens that drew
attention. Each case names one operator and its sizes:

  bounds  kv_history.update_block_bounds: per block of cached tokens the
          smallest and largest value of every key channel
  select  kv_history.select_blocks: the blocks that each run of queries reads,
          by the upper bound of its logits in every block
  sparse  cache_attention.sparse_chunk_attention: attention over those blocks
          and the bf16 tail of the current chunk
  mass    kv_history.key_mass: the attention weight that every cached key drew
  evict   kv_history.evict: the tokens of largest mass, moved to the front of
          another cache

``run`` is the plain form where ``own`` is false (elementary torch operations
in 32 bits, in 64 where values next to a border decide), the framework's calls
where it is true. The widths are the DiT's (24 heads of 128, 10800 tokens a
3 x 45 x 80 chunk, 3600 a latent frame) and those of grouped heads (32 query
heads over 8).
"""
import importlib
import math

import torch

own = False

BF16, F32, F64, FP8 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn
D = 128                # head dim of every attention path
FRAME, CHUNK = 3600, 10800
INF = float("inf")


def _case(kind, name=None, **kw):
    base = dict(kind=kind, B=1, H=24, G=1, Lq=1, kv=0, block=64, q_block=128, fmt="fp8", holes=0.0)
    base.update(kw)
    if name is not None:
        base["name"] = name
    return base


def listed():
    return [
        # eight answers in progress append one token each: the open block of every head
        _case("bounds", "bounds_token", B=8, H=8, start=5000, L=1),
        # a chunk's keys joined the history: the blocks they fall in
        _case("bounds", "bounds_chunk", start=7 * CHUNK, L=CHUNK),
        # one token of eight long answers, four query heads to a cached head
        _case("select", "select_token", B=8, H=8, G=4, Lq=1, q_block=1, kv=131072, top_k=64, first=1, last=2),
        # a denoising pass of a chunk over eight cached ones
        _case("select", "select_chunk", Lq=CHUNK, kv=8 * CHUNK, top_k=128, first=4, last=8),
        # the smallest call: one query over a short history
        _case("sparse", "sparse_one", H=8, Lq=1, q_block=1, kv=4000, top_k=16, Lc=1),
        # one token of eight long answers
        _case("sparse", "sparse_token", B=8, H=8, G=4, Lq=1, q_block=1, kv=131072, top_k=64, Lc=1),
        # a segment's text queries: int8 storage, holes, wide blocks, a ragged history and tail
        _case("sparse", "sparse_text", Lq=777, kv=30011, top_k=24, Lc=777, block=128, q_block=64, fmt="int8", holes=0.02),
        # a denoising pass of a chunk: an eighth of the history and the chunk itself
        _case("sparse", "sparse_chunk", Lq=CHUNK, kv=8 * CHUNK, top_k=128, Lc=CHUNK),
        # what one token of eight answers looked at
        _case("mass", "mass_token", B=8, H=8, G=4, Lq=1, kv=32768),
        # what a latent frame's queries looked at over eight cached chunks
        _case("mass", "mass_frame", Lq=FRAME, kv=8 * CHUNK),
        # a short history halved, its first tokens and its newest kept
        _case("evict", "evict_short", kv=1001, keep=500, first=16, last=64, holes=0.02, fmt="int8"),
        # eight chunks of history cut to four
        _case("evict", "evict_chunks", kv=8 * CHUNK, keep=4 * CHUNK, first=FRAME, last=CHUNK),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["bounds", "select", "sparse", "sparse", "mass", "evict"])
    fmt = rng.choice(["fp8", "fp8", "int8"])
    holes = rng.choice([0.0, 0.0, 0.03])
    H, G = rng.choice([(24, 1), (24, 1), (8, 1), (8, 4), (4, 8), (3, 2)])
    B = rng.choice([1, 1, 2, 4])
    block = rng.choice([64, 64, 128, 256])
    if kind == "bounds":
        L = _log_int(rng, 1, CHUNK // B)
        return _case(kind, B=B, H=H, start=_log_int(rng, 1, 40000), L=L, block=block, fmt=fmt, holes=holes)
    if kind == "evict":
        kv = _log_int(rng, 70, 2 * CHUNK * 4 // B)
        keep = _log_int(rng, 32, max(32, kv * 3 // 4))
        return _case(kind, B=B, H=H, kv=kv, keep=keep, first=min(keep // 4, 16), last=min(keep // 4, 300), fmt=fmt,
                     holes=holes)
    if kind == "mass":
        kv = _log_int(rng, 64, 60000)
        Lq = _log_int(rng, 1, max(1, min(2000, 24 * FRAME * 8 * CHUNK // (kv * B * H * G * 2))))
        return _case(kind, B=B, H=H, G=G, Lq=Lq, kv=kv, fmt=fmt, holes=holes)
    kv = _log_int(rng, 200, 60000)
    Lq = _log_int(rng, 1, max(1, 4000 * 24 // (B * H * G)))
    q_block = rng.choice([1, 16]) if Lq <= 64 else rng.choice([32, 64, 128, 200])
    top_k = min(_log_int(rng, 8, 64), -(-kv // block) + 1)
    if kind == "select":
        return _case(kind, B=B, H=H, G=G, Lq=Lq, kv=kv, block=block, q_block=q_block, top_k=top_k,
                     first=min(1, top_k // 4), last=min(2, top_k // 4), holes=holes)
    return _case(kind, B=B, H=H, G=G, Lq=Lq, kv=kv, block=block, q_block=q_block, top_k=min(top_k, 4096 // block),
                 Lc=rng.choice([0, 1, Lq]), fmt=fmt, holes=holes)


# --------------------------------------------------------------------------
# inputs

def _ceil(a, b):
    return -(-a // b)


def _quantize(x, fmt):
    """Codes and fp32 row scales of the cache formats."""
    amax = x.abs().amax(-1, keepdim=True)
    if fmt == "fp8":
        s = torch.where(amax > 0, amax / 448.0, torch.ones_like(amax))
        return (x / s).to(FP8), s
    s = torch.where(amax > 0, amax / 127.0, torch.ones_like(amax))
    return (x / s).round().clamp(-127, 127).to(torch.int8), s


def _cache(c, cap, g, dev):
    """A cache of keys that resemble their neighbours (a centre per 64 tokens) and values."""
    centre = torch.randn(c["B"], _ceil(cap, 64), c["H"], D, generator=g, device=dev)
    cache = {}
    for key in ("k", "v"):
        x = torch.randn(c["B"], cap, c["H"], D, generator=g, device=dev)
        if key == "k":
            x = 0.8 * x + 0.6 * centre.repeat_interleave(64, dim=1)[:, :cap]
        cache[key], cache[key + "_scale"] = _quantize(x.to(BF16).float(), c["fmt"])
    return cache


def _holes(c, n, g, dev):
    """Which of n tokens are valid (None: all)."""
    return torch.rand(c["B"], n, generator=g, device=dev) >= c["holes"] if c["holes"] else None


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    st = dict(case=c)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev).to(BF16)

    if c["kind"] == "bounds":
        end = c["start"] + c["L"]
        cap = end + 500
        st.update(cache=_cache(c, cap, g, dev), valid=_holes(c, cap, g, dev))
        st["bounds"] = torch.empty(c["B"], _ceil(cap, c["block"]), c["H"], 2, D, dtype=BF16, device=dev)
        st["bounds"][..., 0, :], st["bounds"][..., 1, :] = INF, -INF
        return st
    if c["kind"] == "evict":
        cap = c["kv"] + 300
        st.update(cache=_cache(c, cap, g, dev), valid=_holes(c, cap, g, dev))
        st["mass"] = torch.randn(c["B"], c["H"], c["kv"], generator=g, device=dev).mul(2).exp()
        st["mass"][:, :, -c["kv"] // 8:] = 0  # tokens that no later query has seen yet
        st["out"] = {k: torch.zeros_like(t[:, :c["keep"] + 100]) for k, t in st["cache"].items()}
        return st
    st["q"] = normal(c["B"], c["Lq"], c["H"] * c["G"], D)
    if c["kind"] == "select":
        n = _ceil(c["kv"], c["block"])
        centre = torch.randn(c["B"], n, c["H"], D, generator=g, device=dev)
        spread = torch.rand(c["B"], n, c["H"], D, generator=g, device=dev) + 0.5
        st["bounds"] = torch.stack([centre - spread, centre + spread], dim=3).to(BF16)
        if c["holes"]:  # blocks without a valid token
            gone = torch.rand(c["B"], n, generator=g, device=dev) < c["holes"]
            st["bounds"][:, :, :, 0].masked_fill_(gone[:, :, None, None], INF)
            st["bounds"][:, :, :, 1].masked_fill_(gone[:, :, None, None], -INF)
        return st
    cap = c["kv"] + 200
    st.update(cache=_cache(c, cap, g, dev), valid=_holes(c, cap, g, dev))
    if c["kind"] == "mass":
        st["lse"] = _lse_for(st, c)
        # the masses of a history that was shorter at the last call
        st["prior"] = torch.rand(c["B"], c["H"], c["kv"] * 7 // 8, generator=g, device=dev)
        return st
    n, runs = _ceil(c["kv"], c["block"]), _ceil(c["Lq"], c["q_block"])
    k = min(c["top_k"], n)
    picked = torch.rand(c["B"], c["H"], runs, n, generator=g, device=dev).topk(k, dim=-1).indices.sort(-1).values
    st["idx"] = torch.full((c["B"], c["H"], runs, c["top_k"]), -1, dtype=torch.int32, device=dev)
    st["idx"][..., :k] = picked.int()
    if c["Lc"]:
        st["k_cur"], st["v_cur"] = normal(c["B"], c["Lc"], c["H"], D), normal(c["B"], c["Lc"], c["H"], D)
        st["cur_valid"] = _holes(c, c["Lc"], g, dev)
    return st


def _lse_for(st, c):
    """Row logarithms of the softmax denominators over the cache, a head at a time."""
    rows = torch.empty(c["B"], c["H"] * c["G"], c["Lq"], dtype=F32, device=st["q"].device)
    for h in range(c["H"]):
        k = _values(st["cache"]["k"][:, :c["kv"], h], st["cache"]["k_scale"][:, :c["kv"], h])
        for i in range(c["G"]):
            s = (st["q"][:, :, h * c["G"] + i].float() @ k.transpose(1, 2)) * D ** -0.5
            if st["valid"] is not None:
                s.masked_fill_(~st["valid"][:, None, :c["kv"]], -INF)
            rows[:, h * c["G"] + i] = torch.logsumexp(s, -1)
    return rows


# --------------------------------------------------------------------------
# the operators: plain forms and the framework's calls

def _values(codes, scale):
    """bf16(code * scale), what the cache holds, in 32 bits."""
    return (codes.float() * scale).to(BF16).float()


def _plain_bounds(st, c):
    block, end = c["block"], c["start"] + c["L"]
    j0, j1 = c["start"] // block, _ceil(end, block)
    n = min(j1 * block, st["cache"]["k"].shape[1])
    k = _values(st["cache"]["k"][:, j0 * block:n], st["cache"]["k_scale"][:, j0 * block:n])
    tok = torch.arange(j0 * block, n, device=k.device)
    there = (tok < end)[None, :].expand(c["B"], -1)
    if st["valid"] is not None:
        there = there & st["valid"][:, j0 * block:n]
    there = there[:, :, None, None]
    pad = (0, 0, 0, 0, 0, j1 * block - n)
    lo = torch.nn.functional.pad(torch.where(there, k, INF), pad, value=INF)
    hi = torch.nn.functional.pad(torch.where(there, k, -INF), pad, value=-INF)
    st["bounds"][:, j0:j1, :, 0] = lo.unflatten(1, (-1, block)).amin(2).to(BF16)
    st["bounds"][:, j0:j1, :, 1] = hi.unflatten(1, (-1, block)).amax(2).to(BF16)
    return st["bounds"]


def _plain_select(st, c):
    """In 64 bits, where every sum is exact: a score next to the border decides an index."""
    n, runs, qb = _ceil(c["kv"], c["block"]), _ceil(c["Lq"], c["q_block"]), c["q_block"]
    q = torch.nn.functional.pad(st["q"].double(), (0, 0, 0, 0, 0, runs * qb - c["Lq"]))
    q = q.reshape(c["B"], runs, qb, c["H"], c["G"], D).permute(0, 3, 1, 2, 4, 5)
    up, down = q.clamp_min(0).sum((3, 4)), q.clamp_max(0).sum((3, 4))          # [B, H, runs, D]
    b = st["bounds"][:, :n].double().permute(0, 2, 3, 4, 1)                    # [B, H, 2, D, n]
    gone = (b[:, :, 0, 0] > b[:, :, 1, 0])[:, :, None]                         # [B, H, 1, n]
    b = torch.where(gone[:, :, :, None], 0.0, b)
    score = (up @ b[:, :, 1] + down @ b[:, :, 0]).float()
    j = torch.arange(n, device=q.device)
    score = torch.where((j < c["first"]) | (j >= n - c["last"]), INF, score).masked_fill(gone, -INF)
    best, where = score.sort(dim=-1, descending=True, stable=True)
    k = min(c["top_k"], n)
    where = where[..., :k].masked_fill(best[..., :k] == -INF, n).sort(-1).values
    idx = torch.full((c["B"], c["H"], runs, c["top_k"]), -1, dtype=torch.int32, device=q.device)
    idx[..., :k] = where.masked_fill(where == n, -1).int()
    return idx


def _plain_sparse(st, c):
    B, H, G, qb = c["B"], c["H"], c["G"], c["q_block"]
    runs = st["idx"].shape[2]
    q = torch.nn.functional.pad(st["q"].float(), (0, 0, 0, 0, 0, runs * qb - c["Lq"]))
    q = q.reshape(B, runs, qb, H, G, D).permute(0, 3, 1, 2, 4, 5).flatten(3, 4)      # [B, H, runs, qb G, D]
    dev = q.device
    bi, hi = torch.arange(B, device=dev)[:, None, None, None], torch.arange(H, device=dev)[None, :, None, None]
    listed_ = (st["idx"] >= 0).cumprod(-1).bool()
    tok = st["idx"].clamp_min(0).long()[..., None] * c["block"] + torch.arange(c["block"], device=dev)
    there = (listed_[..., None] & (tok < c["kv"])).flatten(3)
    tok = tok.flatten(3).clamp_max(c["kv"] - 1)                                      # [B, H, runs, keys]
    if st["valid"] is not None:
        there = there & st["valid"][bi, tok]

    def rows(key):
        codes = st["cache"][key]
        got = codes.view(torch.uint8)[bi, tok, hi].view(codes.dtype)
        return _values(got, st["cache"][key + "_scale"][bi, tok, hi])

    s = (q @ rows("k").transpose(3, 4)).masked_fill_(~there[:, :, :, None], -INF)
    if c["Lc"]:
        tail = q.flatten(2, 3) @ st["k_cur"].float().permute(0, 2, 3, 1)
        if st["cur_valid"] is not None:
            tail.masked_fill_(~st["cur_valid"][:, None, None], -INF)
        s = torch.cat([s, tail.unflatten(2, (runs, -1))], dim=-1)
    s.mul_(D ** -0.5)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -INF, 0.0, top)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    keys = tok.shape[-1]
    out = p[..., :keys] @ rows("v")
    if c["Lc"]:
        out = out + (p[..., keys:].flatten(2, 3) @ st["v_cur"].float().permute(0, 2, 1, 3)).unflatten(2, (runs, -1))
    out = torch.where(total > 0, out / total, 0.0).unflatten(3, (qb, G))             # [B, H, runs, qb, G, D]
    out = out.permute(0, 2, 3, 1, 4, 5).reshape(B, runs * qb, H * G, D)[:, :c["Lq"]]
    lse = (top + total.log()).squeeze(-1).unflatten(3, (qb, G)).permute(0, 1, 4, 2, 3)
    return out.to(BF16), lse.reshape(B, H * G, runs * qb)[:, :, :c["Lq"]].contiguous()


def _plain_mass(st, c):
    k = _values(st["cache"]["k"][:, :c["kv"]], st["cache"]["k_scale"][:, :c["kv"]]).permute(0, 2, 3, 1)
    q = st["q"].float().unflatten(2, (c["H"], c["G"])).permute(0, 2, 3, 1, 4).flatten(2, 3)
    lse = st["lse"].unflatten(1, (c["H"], c["G"])).flatten(2, 3)[..., None]
    p = (q @ k).mul_(D ** -0.5).sub_(lse).exp_()
    mass = p.sum(2)
    if st["valid"] is not None:
        mass = mass.masked_fill(~st["valid"][:, None, :c["kv"]], 0.0)
    mass[:, :, :st["prior"].shape[2]] += st["prior"]
    return mass


def _plain_evict(st, c):
    kv, keep = c["kv"], c["keep"]
    t = torch.arange(kv, device=st["mass"].device)
    rank = torch.where((t < c["first"]) | (t >= kv - c["last"]), INF, st["mass"])
    if st["valid"] is not None:
        rank = rank.masked_fill(~st["valid"][:, None, :kv], -INF)
    best, where = rank.sort(dim=-1, descending=True, stable=True)
    where = where[..., :keep].masked_fill(best[..., :keep] == -INF, kv).sort(-1).values
    there = where < kv
    src = where.clamp_max(kv - 1)
    bi, hi = torch.arange(c["B"], device=t.device)[:, None, None], torch.arange(c["H"], device=t.device)[None, :, None]
    for name, out in st["out"].items():
        moved, old = st["cache"][name], out
        if moved.element_size() == 1:
            moved, old = moved.view(torch.uint8), out.view(torch.uint8)
        old = old[:, :keep]
        old.copy_(torch.where(there.transpose(1, 2)[..., None], moved[bi, src, hi].transpose(1, 2), old))
    return where.masked_fill(~there, -1).int(), torch.where(there, st["mass"][bi, hi, src], 0.0)


def _own(st, c):
    hist = importlib.import_module("hy-nomas_amd.kv_history")
    if c["kind"] == "bounds":
        hist.update_block_bounds(st["bounds"], st["cache"], c["start"], c["start"] + c["L"], block=c["block"],
                                 cache_valid=st["valid"])
        return st["bounds"]
    if c["kind"] == "select":
        return hist.select_blocks(st["q"], st["bounds"], c["kv"], c["top_k"], block=c["block"], q_block=c["q_block"],
                                  keep_first=c["first"], keep_last=c["last"])
    if c["kind"] == "sparse":
        ca = importlib.import_module("hy-nomas_amd.cache_attention")
        return ca.sparse_chunk_attention(st["q"], st["cache"], c["kv"], st["idx"], block=c["block"],
                                         q_block=c["q_block"], k_cur=st.get("k_cur"), v_cur=st.get("v_cur"),
                                         cache_valid=st["valid"], cur_valid=st.get("cur_valid"))
    if c["kind"] == "mass":
        return hist.key_mass(st["q"], st["lse"], st["cache"], c["kv"], prior=st["prior"], cache_valid=st["valid"])
    return hist.evict(st["cache"], st["out"], st["mass"], c["kv"], c["keep"], keep_first=c["first"],
                      keep_last=c["last"], cache_valid=st["valid"])


def run(state):
    c = state["case"]
    if own:
        got = _own(state, c)
    else:
        got = {"bounds": _plain_bounds, "select": _plain_select, "sparse": _plain_sparse, "mass": _plain_mass,
               "evict": _plain_evict}[c["kind"]](state, c)
    if c["kind"] == "evict":  # the moved codes as the bytes they are
        out = state["out"]
        return dict(idx=got[0], mass=got[1], k=out["k"].view(torch.uint8), v=out["v"].view(torch.uint8),
                    k_scale=out["k_scale"], v_scale=out["v_scale"])
    return got


# --------------------------------------------------------------------------
# what a pass cannot do without

def work(case):
    c = case
    row = D + 4  # codes and scale of one cached key or value
    q = c["B"] * c["Lq"] * c["H"] * c["G"] * D * 2
    if c["kind"] == "bounds":
        j0, j1 = c["start"] // c["block"], _ceil(c["start"] + c["L"], c["block"])
        keys = c["B"] * c["H"] * (c["start"] + c["L"] - j0 * c["block"])
        return dict(bytes=keys * row + c["B"] * c["H"] * (j1 - j0) * 2 * D * 2, flops=keys * D * 3)
    if c["kind"] == "select":
        n, runs = _ceil(c["kv"], c["block"]), _ceil(c["Lq"], c["q_block"])
        return dict(bytes=q + c["B"] * c["H"] * (n * 2 * D * 2 + runs * c["top_k"] * 4),
                    flops=c["B"] * c["H"] * (runs * n * 4 * D + 2 * c["Lq"] * c["G"] * D))
    if c["kind"] == "sparse":
        runs, k = _ceil(c["Lq"], c["q_block"]), min(c["top_k"], _ceil(c["kv"], c["block"])) * c["block"]
        # a block that several runs of a head list is read once
        seen = min(c["kv"], c["kv"] * (1 - (1 - min(1.0, k / c["kv"])) ** runs))
        rows = c["B"] * c["H"] * c["G"] * c["Lq"]
        return dict(bytes=int(2 * q + rows * 4 + c["B"] * c["H"] * (2 * seen * row + 4 * c["Lc"] * D + runs * c["top_k"] * 4)),
                    flops=rows * (min(k, c["kv"]) + c["Lc"]) * 4 * D)
    if c["kind"] == "mass":
        rows = c["B"] * c["H"] * c["G"] * c["Lq"]
        return dict(bytes=q + rows * 4 + c["B"] * c["H"] * (c["kv"] * (row + 4) + c["kv"] * 7 // 8 * 4),
                    flops=rows * c["kv"] * (2 * D + 3))
    return dict(bytes=c["B"] * c["H"] * (c["kv"] * 4 + c["keep"] * (2 * 2 * row + 3 * 4)), flops=c["B"] * c["H"] * c["kv"])


# --------------------------------------------------------------------------
# 64 bits, from the definitions, head by head

def exact(case, seed):
    c, st = case, prepare(case, seed)
    B, H, G = c["B"], c["H"], c["G"]

    def held(key, b, h, t0, t1):  # what the cache holds of one head's tokens
        x = st["cache"][key][b, t0:t1, h].float() * st["cache"][key + "_scale"][b, t0:t1, h]
        return x.to(BF16).to(F64)

    if c["kind"] == "bounds":
        out = st["bounds"].to(F64)
        end = c["start"] + c["L"]
        for j in range(c["start"] // c["block"], _ceil(end, c["block"])):
            t0, t1 = j * c["block"], min((j + 1) * c["block"], end)
            x = (st["cache"]["k"][:, t0:t1].float() * st["cache"]["k_scale"][:, t0:t1]).to(BF16).to(F64)
            ok = torch.ones(B, t1 - t0, dtype=torch.bool, device=x.device) if st["valid"] is None else st["valid"][:, t0:t1]
            ok = ok[:, :, None, None]
            out[:, j, :, 0] = torch.where(ok, x, INF).min(1).values
            out[:, j, :, 1] = torch.where(ok, x, -INF).max(1).values
        return out
    if c["kind"] in ("select", "evict"):
        return None  # whole numbers and moved values: compared for equality
    scale = 1.0 / math.sqrt(D)
    if c["kind"] == "mass":
        out = torch.zeros(B, H, c["kv"], dtype=F64, device=st["q"].device)
        for b in range(B):
            for h in range(H):
                k = held("k", b, h, 0, c["kv"])
                for i in range(G):
                    for r in range(0, c["Lq"], 1024):
                        q = st["q"][b, r:r + 1024, h * G + i].to(F64)
                        lse = st["lse"][b, h * G + i, r:r + 1024].to(F64)
                        out[b, h] += torch.exp(q @ k.T * scale - lse[:, None]).sum(0)
        if st["valid"] is not None:
            out *= st["valid"][:, None, :c["kv"]]
        out[:, :, :st["prior"].shape[2]] += st["prior"].to(F64)
        return out
    out = torch.zeros(B, c["Lq"], H * G, D, dtype=F64, device=st["q"].device)
    lse = torch.full((B, H * G, c["Lq"]), -INF, dtype=F64, device=st["q"].device)
    if B * H * st["idx"].shape[2] > 6000:
        return None
    lists = st["idx"].cpu().tolist()
    for b in range(B):
        for h in range(H):
            k, v = held("k", b, h, 0, c["kv"]), held("v", b, h, 0, c["kv"])
            ok = torch.ones(c["kv"], dtype=torch.bool, device=k.device) if st["valid"] is None else st["valid"][b, :c["kv"]]
            if c["Lc"]:
                tk, tv = st["k_cur"][b, :, h].to(F64), st["v_cur"][b, :, h].to(F64)
                if st["cur_valid"] is not None:
                    tk, tv = tk[st["cur_valid"][b]], tv[st["cur_valid"][b]]
            for r, blocks in enumerate(lists[b][h]):
                read = torch.tensor([j for j in blocks if j >= 0], device=k.device, dtype=torch.long)
                t = (read[:, None] * c["block"] + torch.arange(c["block"], device=k.device)).flatten()
                t = t[t < c["kv"]]
                t = t[ok[t]]
                keys, vals = k[t], v[t]
                if c["Lc"]:
                    keys, vals = torch.cat([keys, tk]), torch.cat([vals, tv])
                if not len(keys):
                    continue
                r0, r1 = r * c["q_block"], min((r + 1) * c["q_block"], c["Lq"])
                for i in range(G):
                    s = st["q"][b, r0:r1, h * G + i].to(F64) @ keys.T * scale
                    lse[b, h * G + i, r0:r1] = torch.logsumexp(s, -1)
                    out[b, r0:r1, h * G + i] = torch.softmax(s, -1) @ vals
    return out, lse
