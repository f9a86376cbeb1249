"""Operators of the quantized KV cache in pages, as a program calls them.

Roll-outs that branch from one history, and sessions of different lengths, share a
pool of pages: a sequence is a row of page numbers and a length. Each case names one
operator and its sizes:

  write   kv_pages.write_pages: new K/V of every sequence, quantized into its pages
  attend  cache_attention.paged_attention: one new token, drafted ones or a chunk's
          queries over the sequences' pages
  copy    kv_pages.copy_pages: pages copied over all layers (a fork's last pages, a
          compaction's moves)
  read    kv_pages.read_pages: a sequence's keys or values, decoded

``run`` is the plain form where ``own`` is false (elementary torch operations in 32
bits), the framework's calls where it is true. The widths are the DiT's (24 heads of
128, 10800 tokens a 3 x 45 x 80 chunk, 3600 a latent frame, 40 layers) and those of
grouped heads (32 query heads over 8).
"""
import importlib
import math

import torch

own = False

BF16, F32, F64, FP8, I32 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn, torch.int32
D = 128                # head dim of every attention path
FRAME, CHUNK = 3600, 10800
INF = float("inf")


def _case(kind, name=None, **kw):
    base = dict(kind=kind, B=1, H=24, G=1, page=64, fmt="fp8", kv=0, L=1, even=False)
    base.update(kw)
    if name is not None:
        base["name"] = name
    return base


def listed():
    return [
        # one token of each of 64 answers in progress
        _case("write", "write_token", B=64, H=8, kv=8192),
        # text of three sessions, padded to the longest, into the int8 format
        _case("write", "write_text", B=3, kv=5000, L=777, fmt="int8", ragged=True),
        # a chunk's keys and values of two branches, as the projection of all three leaves them
        _case("write", "write_chunk", B=2, kv=2 * CHUNK, L=CHUNK, even=True),
        # the smallest call: one token of one session over a short history
        _case("attend", "attend_one", H=8, kv=700),
        # one token of 32 answers of different lengths, four query heads to a cached head
        _case("attend", "attend_batch", B=32, H=8, G=4, kv=16384),
        # one token of eight long sessions, int8 storage, pages of 256
        _case("attend", "attend_long", B=8, kv=30000, fmt="int8", page=256),
        # five drafted tokens of 16 answers, each row seeing what precedes it
        _case("attend", "attend_draft", B=16, H=8, G=4, L=5, kv=16384, causal=True),
        # a latent frame's queries of two branches over one history and their own frames
        _case("attend", "attend_frame", B=2, L=FRAME, Lc=FRAME, kv=2 * CHUNK, shared=True, even=True),
        # eight branches fork: their half-filled last pages, all layers
        _case("copy", "copy_fork", layers=40, pages=40, pairs=8),
        # half of a pool's pages move to its front
        _case("copy", "copy_compact", layers=40, pages=128, pairs=60, H=16),
        # a short session's keys
        _case("read", "read_short", B=2, kv=900, H=8, fmt="int8"),
        # the history of two branches
        _case("read", "read_chunks", B=2, kv=2 * CHUNK, even=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["write", "write", "attend", "attend", "attend", "copy", "read"])
    fmt = rng.choice(["fp8", "fp8", "int8"])
    page = rng.choice([64, 64, 128, 256])
    H, G = rng.choice([(24, 1), (16, 1), (8, 1), (8, 4), (4, 8), (3, 2)])
    B = rng.choice([1, 2, 3, 8, 17, 40])
    if kind == "copy":
        layers = rng.choice([1, 7, 40])
        pairs = _log_int(rng, 1, max(1, 40 * 60 * 16 * 64 // (layers * H * page)))
        return _case(kind, H=H, page=page, fmt=fmt, layers=layers, pairs=pairs, pages=2 * pairs + rng.randrange(1, 9))
    if kind == "read":
        return _case(kind, B=B, H=H, page=page, fmt=fmt, kv=_log_int(rng, 1, 2 * 2 * CHUNK * 24 // (B * H)),
                     empty=rng.random() < 0.3)
    if kind == "write":
        L = rng.choice([1, _log_int(rng, 2, max(2, 2 * CHUNK * 24 // (B * H)))])
        return _case(kind, B=B, H=H, page=page, fmt=fmt, kv=_log_int(rng, 1, 2 * CHUNK // B), L=L,
                     ragged=rng.random() < 0.5)
    if rng.random() < 0.65:  # a token, or a few
        L = rng.choice([1, 1, 1, rng.randrange(2, 9)])
        return _case(kind, B=B, H=H, G=G, page=page, fmt=fmt, L=L, kv=_log_int(rng, L, 32 * 16384 * 8 // (B * H)),
                     causal=L > 1 and rng.random() < 0.7, empty=L == 1 and rng.random() < 0.3)
    B, L = rng.choice([1, 2, 4]), _log_int(rng, 9, 2000)
    kv = _log_int(rng, L, max(L, min(20000, 24 * FRAME * 2 * CHUNK // (B * H * G * L))))
    causal = rng.random() < 0.3
    Lc = 0 if causal else rng.choice([0, L])
    return _case(kind, B=B, H=H, G=G, page=page, fmt=fmt, L=L, Lc=Lc, kv=kv, causal=causal,
                 shared=rng.random() < 0.3)


# --------------------------------------------------------------------------
# inputs

def _ceil(a, b):
    return -(-a // b)


def _lengths(c):
    """Tokens of each sequence: from ``kv`` down to a tenth of it, in a mixed order."""
    B, kv = c["B"], c["kv"]
    least = c["L"] if c.get("causal") else 0 if c.get("empty") else 1
    if c["even"]:
        return [kv - 37 * b for b in range(B)]
    step = next(s for s in (7, 5, 3, 2, 1) if B % s or B == 1)
    spread = [kv * (1 - 0.9 * (b * step % B) / B) for b in range(B)]
    n = [max(least, round(x)) for x in spread]
    if c.get("empty"):
        n[-1] = 0
    return n


def _counts(c):
    """New tokens of each sequence of a write."""
    if not c.get("ragged"):
        return [c["L"]] * c["B"]
    return [max(0, c["L"] - (c["L"] * b) // c["B"]) for b in range(c["B"])]


def _codes(x, fmt):
    """Codes and fp32 row scales of the cache formats."""
    amax = x.abs().amax(-1, keepdim=True)
    if fmt == "fp8":
        s = torch.where(amax > 0, amax / 448.0, torch.ones_like(amax))
        return (x / s).to(FP8), s
    s = torch.where(amax > 0, amax / 127.0, torch.ones_like(amax))
    q = x / s
    return torch.where(q >= 0, torch.floor(q + 0.5), torch.ceil(q - 0.5)).clamp(-127, 127).to(torch.int8), s


def _pool(c, pages, g, dev):
    """A layer's pool, filled: a page's scales lie head by head."""
    cache = {}
    for key in ("k", "v"):
        x = torch.randn(pages, c["page"], c["H"], D, generator=g, device=dev)
        x *= torch.rand(c["H"], 1, generator=g, device=dev) * 1.5 + 0.5
        cache[key], s = _codes(x.to(BF16).float(), c["fmt"])
        cache[key + "_scale"] = s.transpose(1, 2).contiguous().transpose(1, 2)
    return cache


def _table(c, tokens, g, dev):
    """Page numbers of every sequence for its tokens (int32, -1 behind the last), and
    how many pages the pool has. Shared: the full pages of the shortest are everybody's."""
    need = [_ceil(n, c["page"]) for n in tokens]
    width = max(max(need), 1)
    common = min(n // c["page"] for n in tokens) if c.get("shared") else 0
    pages = common + sum(n - common for n in need) + 3
    order = torch.randperm(pages, generator=g, device=dev).to(I32)
    table = torch.full((c["B"], width), -1, dtype=I32, device=dev)
    at = common
    for b, n in enumerate(need):
        table[b, :common] = order[:common]
        table[b, common:n] = order[at:at + n - common]
        at += n - common
    return table, pages


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    st = dict(case=c)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev).to(BF16)

    if c["kind"] == "copy":
        shape = (c["layers"], c["pages"], c["page"], c["H"])
        st["cache"] = {}
        for key in ("k", "v"):
            x = torch.randint(0, 255, (*shape, D), generator=g, device=dev, dtype=torch.uint8)
            st["cache"][key] = x.view(FP8 if c["fmt"] == "fp8" else torch.int8)
            s = torch.rand(c["layers"], c["pages"], c["H"], c["page"], 1, generator=g, device=dev)
            st["cache"][key + "_scale"] = s.transpose(2, 3)
        order = torch.randperm(c["pages"], generator=g, device=dev).tolist()
        st["src"], st["dst"] = order[:c["pairs"]], order[c["pairs"]:2 * c["pairs"]]
        st["src_dev"], st["dst_dev"] = torch.tensor(st["src"], device=dev), torch.tensor(st["dst"], device=dev)
        return st
    n = _lengths(c)
    if c["kind"] == "write":
        counts = _counts(c)
        table, pages = _table(c, [a + b for a, b in zip(n, counts)], g, dev)
        # q, k and v of one projection: the rows of k and v lie apart
        qkv = normal(c["B"], c["L"], 3, c["H"], D)
        st.update(cache=_pool(c, pages, g, dev), table=table, start=torch.tensor(n, dtype=I32, device=dev),
                  k=qkv[:, :, 1], v=qkv[:, :, 2], status=torch.zeros(1, dtype=I32, device=dev),
                  counts=torch.tensor(counts, dtype=I32, device=dev) if c.get("ragged") else None)
        return st
    table, pages = _table(c, n, g, dev)
    st.update(cache=_pool(c, pages, g, dev), table=table, kv_len=torch.tensor(n, dtype=I32, device=dev))
    if c["kind"] == "attend":
        st["q"] = normal(c["B"], c["L"], c["H"] * c["G"], D)
        if c.get("Lc"):
            st["k_cur"], st["v_cur"] = normal(c["B"], c["Lc"], c["H"], D), normal(c["B"], c["Lc"], c["H"], D)
    return st


# --------------------------------------------------------------------------
# the operators: plain forms and the framework's calls

def _raw(t):
    return t.view(torch.uint8)


def _plain_write(st, c):
    ok = torch.isfinite(st["k"]).all() & torch.isfinite(st["v"]).all()
    st["status"].copy_((~ok).to(I32))
    t = torch.arange(c["L"], device=st["k"].device)
    pos = (st["start"][:, None] + t).long()
    page = st["table"].gather(1, (pos // c["page"]).clamp_max(st["table"].shape[1] - 1)).long()
    there = torch.ones_like(pos, dtype=torch.bool) if st["counts"] is None else t < st["counts"][:, None]
    page, slot = page[there], (pos % c["page"])[there]
    for key in ("k", "v"):
        codes, s = _codes(st[key].float(), c["fmt"])
        old, old_s = _raw(st["cache"][key]), st["cache"][key + "_scale"]
        old[page, slot] = torch.where(ok, _raw(codes)[there], old[page, slot])
        old_s[page, slot] = torch.where(ok, s[there], old_s[page, slot])
    return st["status"]


def _rows(st, c, key, tokens):
    """What the cache holds of the first ``tokens`` tokens of every sequence, in 32
    bits [B, tokens, H, D]; zeros past a sequence's end."""
    t = torch.arange(tokens, device=st["table"].device)
    there = t < st["kv_len"][:, None]
    page = st["table"][:, t // c["page"]].clamp_min(0).long()
    codes = st["cache"][key]
    x = _raw(codes)[page, t % c["page"]].view(codes.dtype).float()
    x = (x * st["cache"][key + "_scale"][page, t % c["page"]]).to(BF16).float()
    return x.masked_fill_(~there[:, :, None, None], 0.0)


def _plain_read(st, c):
    return _rows(st, c, "k", c["kv"]).to(BF16)


def _plain_attend(st, c):
    B, H, G, L, kv = c["B"], c["H"], c["G"], c["L"], st["table"].shape[1] * c["page"]
    dev = st["q"].device
    q = st["q"].float().reshape(B, L, H, G, D).permute(0, 2, 1, 3, 4).flatten(2, 3)          # [B, H, L G, D]
    k, v = (_rows(st, c, key, kv).transpose(1, 2) for key in ("k", "v"))                     # [B, H, kv, D]
    if c.get("Lc"):
        k = torch.cat([k, st["k_cur"].float().transpose(1, 2)], dim=2)
        v = torch.cat([v, st["v_cur"].float().transpose(1, 2)], dim=2)
    t = torch.arange(kv, device=dev)
    end = st["kv_len"][:, None]                                                              # [B, 1 or L]
    if c.get("causal"):
        end = end - (L - 1) + torch.arange(L, device=dev)
    gone = t >= end[:, :, None]                                                              # [B, 1 or L, kv]
    if c.get("causal"):
        gone = gone.repeat_interleave(G, dim=1)
    s = q @ k.transpose(2, 3).contiguous()
    s[..., :kv].masked_fill_(gone[:, None], -INF)
    s.mul_(D ** -0.5)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -INF, 0.0, top)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.where(total > 0, (p @ v.contiguous()) / total, 0.0)
    out = out.unflatten(2, (L, G)).permute(0, 2, 1, 3, 4).reshape(B, L, H * G, D)
    lse = (top + total.log()).squeeze(-1).unflatten(2, (L, G)).transpose(2, 3).reshape(B, H * G, L)
    return out.to(BF16), lse


def _plain_copy(st, c):
    for x in st["cache"].values():
        x = _raw(x) if x.element_size() == 1 else x
        x[:, st["dst_dev"]] = x[:, st["src_dev"]]


def _own(st, c):
    pages = importlib.import_module("hy-nomas_amd.kv_pages")
    if c["kind"] == "write":
        pages.write_pages(st["cache"], st["k"], st["v"], st["table"], st["start"], counts=st["counts"],
                          status=st["status"], gpu_scales=True)
        return st["status"]
    if c["kind"] == "copy":
        return pages.copy_pages(st["cache"], st["src"], st["dst"])
    if c["kind"] == "read":
        return pages.read_pages(st["cache"], "k", st["table"], st["kv_len"], c["kv"])
    ca = importlib.import_module("hy-nomas_amd.cache_attention")
    return ca.paged_attention(st["q"], st["cache"], st["table"], st["kv_len"], causal=c.get("causal", False),
                              k_cur=st.get("k_cur"), v_cur=st.get("v_cur"))


def run(state):
    c = state["case"]
    if own:
        got = _own(state, c)
    else:
        got = {"write": _plain_write, "attend": _plain_attend, "copy": _plain_copy, "read": _plain_read}[c["kind"]](state, c)
    if c["kind"] == "write":
        return dict(state["cache"], status=got)
    if c["kind"] == "copy":  # the moved codes as the bytes they are
        return {n: _raw(x) if x.element_size() == 1 else x for n, x in state["cache"].items()}
    return got


# --------------------------------------------------------------------------
# what a pass cannot do without

def work(case):
    c = case
    row = D + 4  # codes and scale of one cached key or value
    if c["kind"] == "copy":
        return dict(bytes=2 * 2 * c["layers"] * c["pairs"] * c["page"] * c["H"] * row, flops=0)
    if c["kind"] == "write":
        rows = 2 * sum(_counts(c)) * c["H"]
        return dict(bytes=rows * (2 * D + row), flops=rows * 3 * D)
    n = _lengths(c)
    if c["kind"] == "read":  # rows past a sequence's end are written too
        return dict(bytes=c["H"] * (sum(n) * row + c["B"] * c["kv"] * 2 * D), flops=c["H"] * sum(n) * D)
    common = min(n) // c["page"] * c["page"] if c.get("shared") else 0
    keys = common + sum(x - common for x in n)  # pages that several sequences share are read once
    rows = c["H"] * c["G"] * c["L"]
    Lc = c.get("Lc", 0)
    seen = sum(x - (c["L"] - 1) / 2 if c.get("causal") else x for x in n) + c["B"] * Lc
    return dict(bytes=int(c["H"] * (2 * keys * row + 2 * c["B"] * Lc * 2 * D) + c["B"] * rows * (2 * 2 * D + 4)),
                flops=int(rows * seen * 4 * D))


# --------------------------------------------------------------------------
# 64 bits, from the definitions, sequence by sequence

def exact(case, seed):
    c, st = case, prepare(case, seed)
    if c["kind"] == "copy":
        return None  # moved values: compared for equality
    table = st["table"].tolist()
    if c["kind"] == "write":
        out, most = {}, 448.0 if c["fmt"] == "fp8" else 127.0
        for key in ("k", "v"):
            codes = st["cache"][key].to(F64)
            scale = st["cache"][key + "_scale"].to(F64)
            for b, n in enumerate(_counts(c)):
                t = st["start"][b].item() + torch.arange(n, device=codes.device)
                page = torch.tensor(table[b], device=codes.device)[t // c["page"]]
                x = st[key][b, :n].to(F64)
                s = x.abs().max(-1, keepdim=True).values / most
                codes[page, t % c["page"]] = x / s
                scale[page, t % c["page"]] = s
            out[key], out[key + "_scale"] = codes if c["fmt"] == "fp8" else None, scale
        return dict(out, status=None)
    n = st["kv_len"].tolist()

    def held(key, b, h):  # what the cache holds of one head of a sequence
        t = torch.arange(n[b], device=st["table"].device)
        page = torch.tensor(table[b], device=t.device)[t // c["page"]].long()
        codes, scale = st["cache"][key][:, :, h].float(), st["cache"][key + "_scale"][:, :, h]
        return (codes[page, t % c["page"]] * scale[page, t % c["page"]]).to(BF16).to(F64)

    B, H, G, L = c["B"], c["H"], c["G"], c["L"]
    dev = st["table"].device
    if c["kind"] == "read":
        out = torch.zeros(B, c["kv"], H, D, dtype=F64, device=dev)
        for b in range(B):
            for h in range(H):
                out[b, :n[b], h] = held("k", b, h)
        return out
    if B * H > 2000:
        return None
    out = torch.zeros(B, L, H * G, D, dtype=F64, device=dev)
    lse = torch.full((B, H * G, L), -INF, dtype=F64, device=dev)
    for b in range(B):
        for h in range(H):
            keys, vals = held("k", b, h), held("v", b, h)
            if c.get("Lc"):
                keys = torch.cat([keys, st["k_cur"][b, :, h].to(F64)])
                vals = torch.cat([vals, st["v_cur"][b, :, h].to(F64)])
            if not len(keys):
                continue
            for i in range(G):
                s = st["q"][b, :, h * G + i].to(F64) @ keys.T / math.sqrt(D)
                if c.get("causal"):
                    later = torch.arange(len(keys), device=dev) > n[b] - L + torch.arange(L, device=dev)[:, None]
                    s = s.masked_fill(later, -INF)
                lse[b, h * G + i] = torch.logsumexp(s, -1)
                out[b, :, h * G + i] = torch.softmax(s, -1) @ vals
    return out, lse
