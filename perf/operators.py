"""The attention side of a serving step on one GPU, as cases that can be timed and compared: the
root-mean-square norm with the residual's addition and an 8-bit output, rotary positions, the paged
8-bit key/value cache as it is written and read back, and attention over that cache.

``listed()`` spans the range of each operator, ``draw(rng)`` gives another case of the same ranges.
``run`` makes one pass: in elementary torch operations in 32 bits, or through the package's entry
points where ``own`` is true.  ``exact`` is the same result from the definition in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

HEAD = 128            # head dimension of the attention kernels
EPS = 1e-6
E4M3 = 448.0          # largest finite e4m3 value
E_MIN, E_MAX = -120, 120
BASE = 10000.0
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # Norm before a projection in a decode step of 16 sequences: the smallest call, latency counts.
        dict(name="norm_decode", path="norm", rows=16, d=8192, dtype="bf16", residual=True, strided=False),
        # The norm of the benchmark's prefill step, feeding the block-scaled fp8 linear.
        dict(name="norm_quant_prefill", path="norm_quant", rows=8192, d=8192, dtype="bf16", residual=True,
             pow2=True),
        # Its backward pass on a training batch at the expert layer's width, with the gradient that
        # comes down the residual stream.
        dict(name="norm_backward", path="norm_bwd", rows=4096, d=7168, dtype="bf16", dh=True),
        # Rotary positions of a context-parallel rank's queries and keys.
        dict(name="rope_prefill", path="rope", b=1, s=16384, hq=32, hkv=8, dim=128, rot=128, dtype="bf16",
             interleaved=False, scaling="none", inverse=False),
        # The gradient of a scaled rotation of half of the head, interleaved pairs, ragged length.
        dict(name="rope_backward_partial", path="rope", b=2, s=2047, hq=16, hkv=16, dim=128, rot=64,
             dtype="bf16", interleaved=True, scaling="yarn", inverse=True),
        # What a decode step writes: one token for each of 32 sequences of different lengths, queries
        # rotated in the same call; the last page of each is read back.
        dict(name="append_decode", path="append", b=32, s=1, ctx=6001, hq=32, hkv=8, page=64,
             interleaved=False, rot=128),
        # A prompt of no round length behind a cached prefix is written and read back.
        dict(name="append_prefill", path="append", b=2, s=8001, ctx=777, hq=32, hkv=8, page=64,
             interleaved=False, rot=128),
        # One sequence on one of eight tensor-parallel ranks: latency of a short context.
        dict(name="attend_decode_one", path="attend", b=1, s=1, ctx=777, hq=8, hkv=1, page=64, window=0,
             sinks=0, ragged=False),
        # The decode shape of the attention kernels, from the cache: 16 sequences, about 6001 tokens each.
        dict(name="attend_decode", path="attend", b=16, s=1, ctx=6001, hq=32, hkv=8, page=64, window=0,
             sinks=0, ragged=True),
        # Long contexts under a sliding window with four tokens that stay visible, four tokens a step
        # (draft and verify), small pages.
        dict(name="attend_verify_window", path="attend", b=32, s=4, ctx=16384, hq=64, hkv=8, page=16,
             window=4096, sinks=4, ragged=True),
        # Chunked prefill: a ragged chunk of queries behind a cached prefix.
        dict(name="attend_chunk", path="attend", b=1, s=1000, ctx=7000, hq=32, hkv=8, page=64, window=0,
             sinks=0, ragged=False),
        # A whole prompt under a sliding window.
        dict(name="attend_prefill_window", path="attend", b=1, s=8192, ctx=8192, hq=32, hkv=8, page=64,
             window=2048, sinks=4, ragged=False),
    ]


def _log_int(rng, lo, hi, mult=1):
    """An integer of [lo, hi], spread over its logarithm, a multiple of ``mult``."""
    x = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(max(x // mult * mult, lo), hi)


def draw(rng):
    path = rng.choice(["norm", "norm_quant", "norm_bwd", "rope", "append", "attend", "attend", "attend"])
    if path == "norm":
        return dict(path=path, rows=_log_int(rng, 1, 8192), d=_log_int(rng, 64, 8192),
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), residual=rng.random() < 0.7,
                    strided=rng.random() < 0.3)
    if path == "norm_quant":
        return dict(path=path, rows=_log_int(rng, 1, 8192), d=_log_int(rng, 128, 8192, 128),
                    dtype=rng.choice(["bf16", "bf16", "fp16"]), residual=rng.random() < 0.7,
                    pow2=rng.random() < 0.6)
    if path == "norm_bwd":
        return dict(path=path, rows=_log_int(rng, 1, 8192), d=_log_int(rng, 64, 8192),
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), dh=rng.random() < 0.6)
    if path == "rope":
        dim = rng.choice([64, 128, 128, 192])
        hkv = rng.choice([1, 2, 8])
        return dict(path=path, b=rng.choice([1, 2, 3]), s=_log_int(rng, 1, 5000), hq=hkv * rng.choice([1, 4]),
                    hkv=hkv, dim=dim, rot=rng.choice([dim, dim // 2, dim // 2 + 2]),
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), interleaved=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "ntk", "yarn"]), inverse=rng.random() < 0.4)
    hkv = rng.choice([1, 2, 4, 8])
    page = rng.choice([16, 32, 64, 64, 128])
    if path == "append":
        if rng.random() < 0.5:
            b, s = _log_int(rng, 1, 64), rng.choice([1, 1, 2, 4])
        else:
            b, s = rng.choice([1, 2, 3]), _log_int(rng, 16, 5000)
        return dict(path=path, b=b, s=s, ctx=_log_int(rng, 1, 4096) - 1, hq=hkv * rng.choice([1, 4, 8]),
                    hkv=hkv, page=page, interleaved=rng.random() < 0.4, rot=rng.choice([128, 128, 64]))
    windowed = rng.random() < 0.4
    window, sinks = (_log_int(rng, 64, 4096), rng.choice([0, 1, 4, 130])) if windowed else (0, 0)
    if rng.random() < 0.6:                       # decode, a few query tokens at most
        return dict(path=path, b=_log_int(rng, 1, 32), s=rng.choice([1, 1, 1, 2, 4, 8]),
                    ctx=_log_int(rng, 16, 16384), hq=hkv * rng.choice([1, 3, 4, 8]), hkv=hkv, page=page,
                    window=window, sinks=sinks, ragged=rng.random() < 0.7)
    s = _log_int(rng, 16, 4096)
    return dict(path=path, b=rng.choice([1, 2]), s=s, ctx=s + rng.choice([0, 0, 333, 4096]),
                hq=hkv * rng.choice([1, 4]), hkv=hkv, page=page, window=window, sinks=sinks,
                ragged=rng.random() < 0.5)


class _State:
    """What a program holds between calls."""

    def __init__(self, **kw):
        self.__dict__.update(kw)


# ------------------------------------------------------------------------------------ inputs
def _lengths(case):
    """Tokens of each sequence, the new ones included: the longest has ``ctx``, the others down to half."""
    b, ctx, s = case["b"], case["ctx"], case["s"]
    if not case.get("ragged", True):
        return [ctx] * b
    return [max(s, ctx - (i * ctx) // (2 * b)) for i in range(b)]


def _frequencies(rot, scaling):
    """Angle per position of each pair (64 bits) and the factor on cos and sin."""
    i = torch.arange(0, rot, 2, dtype=torch.float64) / rot
    if scaling == "ntk":                        # the base stretched so that the lowest frequency is / 4
        return (BASE * 4.0 ** (rot / max(rot - 2, 1))) ** -i, 1.0
    f = BASE ** -i
    if scaling == "linear":
        return f / 4.0, 1.0
    if scaling == "yarn":                       # factor 4 over 4096 positions, by parts
        def dim_of(turns):
            return rot * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(BASE))

        lo, hi = max(math.floor(dim_of(32)), 0), min(math.ceil(dim_of(1)), rot - 1)
        ramp = ((torch.arange(rot // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return f * (1 - ramp) + f / 4.0 * ramp, 0.1 * math.log(4.0) + 1.0
    return f, 1.0


def _scaling_argument(scaling):
    return {"none": None, "linear": dict(kind="linear", factor=4.0), "ntk": dict(kind="ntk", factor=4.0),
            "yarn": dict(kind="yarn", factor=4.0, original_positions=4096)}[scaling]


def _raw(case, seed):
    """The tensors of a case, the same for every form of it."""
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    path = case["path"]

    def randn(*shape, dtype=torch.bfloat16, scale=1.0):
        return (torch.randn(*shape, device=dev, generator=g) * scale).to(dtype)

    if path.startswith("norm"):
        rows, d, dt = case["rows"], case["d"], DTYPES[case["dtype"]]
        # a residual stream: rows of different size, some columns far above the rest
        gain = torch.exp(0.5 * torch.randn(rows, 1, device=dev, generator=g))
        col = 1.0 + 8.0 * (torch.rand(1, d, device=dev, generator=g) < 0.01)
        w = (1.0 + 0.1 * torch.randn(d, device=dev, generator=g)).to(dt)
        x = (torch.randn(rows, d, device=dev, generator=g) * gain * col).to(dt)
        r = dict(w=w, x=x)
        if path == "norm_bwd":
            r["dy"] = randn(rows, d, dtype=dt)
            r["dh"] = randn(rows, d, dtype=dt) if case["dh"] else None
            return r
        if case.get("strided"):                 # the rows are part of a wider tensor
            wide = torch.zeros(rows, d + 24, dtype=dt, device=dev)
            wide[:, 8:8 + d] = x
            r["x"] = wide[:, 8:8 + d]
        r["res"] = (torch.randn(rows, d, device=dev, generator=g) * gain).to(dt) if case["residual"] else None
        return r
    if path == "rope":
        b, s, hq, hkv, dim, dt = (case[x] for x in ("b", "s", "hq", "hkv", "dim", "dtype"))
        x = randn(b, s, hq + hkv, dim, dtype=DTYPES[dt])     # a fused projection's queries and keys
        first = torch.randint(0, 4096, (b, 1), device=dev, generator=g)
        return dict(q=x[:, :, :hq], k=x[:, :, hq:], pos=(first + torch.arange(s, device=dev)).int())
    b, s, hq, hkv, page = (case[x] for x in ("b", "s", "hq", "hkv", "page"))
    if path == "append":
        start = [n for n in _lengths(dict(case, s=0))]
        total = max(start) + s
    else:
        lens = _lengths(case)
        start = [n - s for n in lens]
        total = max(lens)
    cols = (total + page - 1) // page
    pages = torch.randperm(b * cols, device=dev, generator=g).int().view(b, cols)
    # keys with channels of different size, as rotary models have them; a few large tokens
    ch = torch.exp(0.7 * torch.randn(2, 1, 1, hkv, HEAD, device=dev, generator=g))
    have = max(start) if path == "append" else total
    kv = torch.randn(2, b, have, hkv, HEAD, device=dev, generator=g) * ch
    kv = kv.bfloat16()
    r = dict(start=torch.tensor(start, dtype=torch.int32, device=dev), pages=pages, kv=kv, total=total,
             q=randn(b, s, hq, HEAD))
    if path == "append":
        new = torch.randn(2, b, s, hkv, HEAD, device=dev, generator=g) * ch
        new = new * (1.0 + 3.0 * (torch.rand(1, b, s, 1, 1, device=dev, generator=g) < 0.05))
        r["new"] = new.bfloat16()
        r["valid"] = r["start"]
    else:
        r["valid"] = r["start"] + s
    return r


def _exponent(amax):
    """The smallest e with amax * 2^-e <= 448."""
    m, x = torch.frexp(amax)
    e = x - 9 + (m > 0.875).int()
    return torch.where(amax > 0, e, torch.full_like(e, E_MIN)).clamp(E_MIN, E_MAX)


def _pow2(e):
    return torch.exp2(e.float())


def _blocks(kv, valid, page):
    """Dense [2, B, T, H, 128] -> e4m3 [2, B, P, page, H, 128] with exponents [2, B, P, H]; tokens from
    ``valid`` on are zero."""
    n, b, t, h, d = kv.shape
    pad = (-t) % page
    x = torch.nn.functional.pad(kv.float(), (0, 0, 0, 0, 0, pad))
    seen = torch.arange(t + pad, device=kv.device)[None, :] < valid[:, None]
    x = (x * seen[None, :, :, None, None]).view(n, b, -1, page, h, d)
    e = _exponent(x.abs().amax(dim=(3, 5)))
    q = (x * _pow2(-e)[:, :, :, None, :, None]).clamp(-E4M3, E4M3).to(torch.float8_e4m3fn)
    return q, e


def prepare(case, seed):
    r = _raw(case, seed)
    path = case["path"]
    dev = torch.device("cuda", torch.cuda.current_device())
    if path.startswith("norm"):
        return _State(case=case, **r)
    if path == "rope" or path == "append":
        f, m = _frequencies(case["rot"], case.get("scaling", "none"))
        top = 4096 + case["s"] + case.get("ctx", 0)
        if own:
            from commbench_b200.ops.rope import RopeTable

            r["table"] = RopeTable(case["rot"], top, base=BASE, interleaved=case["interleaved"],
                                   scaling=_scaling_argument(case.get("scaling", "none")), device=dev)
        else:
            angle = torch.arange(top, dtype=torch.float64, device=dev)[:, None] * f.to(dev)
            r["cos"], r["sin"] = (torch.cos(angle) * m).float(), (torch.sin(angle) * m).float()
        if path == "rope":
            return _State(case=case, **r)
    page, kv, valid = case["page"], r.pop("kv"), r.pop("valid")
    pool = r["pages"].numel()
    if own:
        from commbench_b200.ops.kvcache import KVCache8

        cache = KVCache8(pool, case["hkv"], page=page, device=dev)
        if kv.shape[2] > 0:
            cache.append(kv[0], kv[1], r["pages"], torch.zeros_like(valid), count=valid)
        return _State(case=case, cache=cache, **r)
    # the same content as plain arrays: [page, key or value, token, head, 128] and [page, key or value, head]
    data = torch.zeros(pool, 2, page, case["hkv"], HEAD, dtype=torch.float8_e4m3fn, device=dev)
    exps = torch.full((pool, 2, case["hkv"]), E_MIN, dtype=torch.int32, device=dev)
    if kv.shape[2] > 0:
        q, e = _blocks(kv, valid, page)
        ids = r["pages"][:, :q.shape[2]].long()
        data.view(torch.uint8)[ids] = q.view(torch.uint8).permute(1, 2, 0, 3, 4, 5)
        exps[ids] = e.permute(1, 2, 0, 3)
    return _State(case=case, data=data, exps=exps, **r)


# --------------------------------------------------------------------------------------- run
def run(s):
    path = s.case["path"]
    if own:
        return _OWN[path](s)
    return _PLAIN[path](s)


def _own_norm(s):
    from commbench_b200.ops.norm import rms_norm

    return rms_norm(s.x, s.w, residual=s.res, eps=EPS)


def _own_norm_quant(s):
    from commbench_b200.ops.gemm import dequantize_blockscaled
    from commbench_b200.ops.norm import rms_norm_quant

    out = rms_norm_quant(s.x, s.w, residual=s.res, eps=EPS, pow2=s.case["pow2"])
    y = dequantize_blockscaled(out[0], out[1], 1)
    return (y, out[-1]) if s.res is not None else y


def _own_norm_bwd(s):
    from commbench_b200.ops.norm import rms_norm_backward

    return rms_norm_backward(s.dy, s.x, s.w, dh=s.dh, eps=EPS)


def _own_rope(s):
    from commbench_b200.ops.rope import rope

    return rope((s.q, s.k), s.pos, s.table, inverse=s.case["inverse"])


def _own_append(s):
    c = s.case
    q = s.cache.append(s.new[0], s.new[1], s.pages, s.start, rope=s.table, q=s.q)
    k, v = s.cache.read(s.pages, s.start - (c["page"] - 1), c["s"] + c["page"] - 1)
    return q, k, v


def _own_attend(s):
    c = s.case
    return s.cache.attend(s.q, s.pages, s.start, window=c["window"], sinks=c["sinks"], max_len=s.total)


def _plain_rms(s):
    x = s.x.float() if s.res is None else s.x.float() + s.res.float()
    return x, x * torch.rsqrt((x * x).mean(dim=1, keepdim=True) + EPS) * s.w.float()


def _plain_norm(s):
    h, y = _plain_rms(s)
    y = y.to(s.x.dtype)
    return y if s.res is None else (y, h.to(s.x.dtype))


def _plain_norm_quant(s):
    h, y = _plain_rms(s)
    b = y.view(y.shape[0], -1, 128)
    amax = b.abs().amax(dim=2, keepdim=True)
    sc = torch.where(amax > 0, amax / torch.full_like(amax, E4M3), torch.ones_like(amax))
    if s.case["pow2"]:
        m, e = torch.frexp(sc)
        sc = _pow2(torch.where(m > 0.5, e, e - 1))
    q = (b * (1.0 / sc)).clamp(-E4M3, E4M3).to(torch.float8_e4m3fn)
    y = (q.float() * sc).view_as(y).bfloat16()
    return y if s.res is None else (y, h.to(s.x.dtype))


def _plain_norm_bwd(s):
    h, dy = s.x.float(), s.dy.float()
    rstd = torch.rsqrt((h * h).mean(dim=1, keepdim=True) + EPS)
    g = dy * s.w.float()
    dx = rstd * (g - h * rstd * rstd * (g * h).mean(dim=1, keepdim=True))
    if s.dh is not None:
        dx = dx + s.dh.float()
    return dx.to(s.x.dtype), (dy * h * rstd).sum(dim=0)


def _rotate(x, cos, sin, rot, interleaved, inverse=False):
    """x [..., H, D] (32 or 64 bits), cos / sin [..., 1, rot / 2]."""
    sin = -sin if inverse else sin
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    ya, yb = a * cos - b * sin, b * cos + a * sin
    y = torch.stack((ya, yb), dim=-1).flatten(-2) if interleaved else torch.cat((ya, yb), dim=-1)
    return torch.cat((y, x[..., rot:]), dim=-1)


def _plain_rope(s):
    c = s.case
    cos, sin = s.cos[s.pos.long()][:, :, None], s.sin[s.pos.long()][:, :, None]
    return tuple(_rotate(x.float(), cos, sin, c["rot"], c["interleaved"], c["inverse"]).to(x.dtype)
                 for x in (s.q, s.k))


def _plain_append(s):
    c = s.case
    page, n = c["page"], c["s"]
    pos = s.start[:, None].long() + torch.arange(n, device=s.start.device)
    cos, sin = s.cos[pos][:, :, None], s.sin[pos][:, :, None]
    q = _rotate(s.q.float(), cos, sin, c["rot"], c["interleaved"]).bfloat16()
    new = torch.stack((_rotate(s.new[0].float(), cos, sin, c["rot"], c["interleaved"]), s.new[1].float()))
    # the pages that new tokens fall into, as values, with the new tokens in place
    first = s.start.long() // page
    cols = first[:, None] + torch.arange((n + page - 2) // page + 1, device=first.device)
    inside = cols < s.pages.shape[1]
    ids = s.pages.gather(1, cols.clamp(max=s.pages.shape[1] - 1)).long()
    t = cols[:, :, None] * page + torch.arange(page, device=first.device)         # [B, P, page]
    i = t - s.start[:, None, None]
    is_new = ((i >= 0) & (i < n) & inside[:, :, None])[:, :, None, :, None, None]
    had = s.start[:, None] > cols * page                                            # older tokens in the page
    picked = new[:, torch.arange(c["b"], device=t.device)[:, None, None], i.clamp(0, n - 1)]
    picked = picked.permute(1, 2, 0, 3, 4, 5)                                       # [B, P, 2, page, H, 128]
    e_old = s.exps[ids]
    old = s.data.view(torch.uint8)[ids].view(torch.float8_e4m3fn).float() * _pow2(e_old)[:, :, :, None, :, None]
    e = _exponent((picked.abs() * is_new).amax(dim=(3, 5)))
    e = torch.where(had[:, :, None, None], torch.maximum(e, e_old), e)
    keep = is_new | (t < s.start[:, None, None])[:, :, None, :, None, None]
    x = torch.where(is_new, picked, old) * keep * _pow2(-e)[:, :, :, None, :, None]
    x = x.clamp(-E4M3, E4M3).to(torch.float8_e4m3fn).view(torch.uint8)
    touched = inside & (cols * page < s.start[:, None] + n)
    s.data.view(torch.uint8)[ids[touched]] = x[touched]
    s.exps[ids[touched]] = e[touched]
    # the new tokens and the page - 1 before them
    r = s.start[:, None].long() - (page - 1) + torch.arange(n + page - 1, device=first.device)
    at = s.pages.gather(1, (r.clamp(min=0) // page)).long()
    v = s.data.view(torch.uint8)[at, :, r.clamp(min=0) % page].view(torch.float8_e4m3fn).float()
    v = v * _pow2(s.exps[at])[..., None] * (r >= 0)[:, :, None, None, None]
    return q, v[:, :, 0].bfloat16(), v[:, :, 1].bfloat16()


def _plain_attend(s):
    c = s.case
    b, n, hq, hkv = c["b"], c["s"], c["hq"], c["hkv"]
    ids = s.pages.long()
    kv = s.data.view(torch.uint8)[ids].view(torch.float8_e4m3fn).float()          # [B, P, 2, page, H, 128]
    kv = kv * _pow2(s.exps[ids])[:, :, :, None, :, None]
    k, v = kv.permute(2, 0, 4, 1, 3, 5).reshape(2, b, hkv, -1, HEAD)
    q = s.q.float().view(b, n, hkv, hq // hkv, HEAD).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, HEAD)
    x = (q @ k.transpose(-1, -2) / math.sqrt(HEAD)).view(b, hkv, hq // hkv, n, -1)
    p = (s.start[:, None] + torch.arange(n, device=q.device))[:, None, None, :, None]
    j = torch.arange(x.shape[-1], device=q.device)
    seen = j <= p
    if c["window"]:
        seen = seen & ((j > p - c["window"]) | (j < c["sinks"]))
    x = x.masked_fill(~seen, float("-inf"))
    m = x.amax(dim=-1, keepdim=True).clamp(min=-3e38)
    w = torch.exp(x - m)
    total = w.sum(dim=-1, keepdim=True)
    o = (w.view(b, hkv, -1, x.shape[-1]) @ v).view(b, hkv, hq // hkv, n, HEAD)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse = (m + torch.log(total)).squeeze(-1).reshape(b, hq, n)
    return o.permute(0, 3, 1, 2, 4).reshape(b, n, hq, HEAD).bfloat16(), lse


_OWN = {"norm": _own_norm, "norm_quant": _own_norm_quant, "norm_bwd": _own_norm_bwd, "rope": _own_rope,
        "append": _own_append, "attend": _own_attend}
_PLAIN = {"norm": _plain_norm, "norm_quant": _plain_norm_quant, "norm_bwd": _plain_norm_bwd,
          "rope": _plain_rope, "append": _plain_append, "attend": _plain_attend}


# -------------------------------------------------------------------------------------- work
def work(case):
    path = case["path"]
    if path.startswith("norm"):
        n, d = case["rows"] * case["d"], case["d"]
        sz = 4 if case["dtype"] == "fp32" else 2
        if path == "norm":
            return {"bytes": n * sz * (4 if case["residual"] else 2) + d * sz, "flops": 4 * n}
        if path == "norm_quant":
            return {"bytes": n * (sz * (3 if case["residual"] else 1) + 2) + d * sz, "flops": 7 * n}
        return {"bytes": n * sz * (4 if case["dh"] else 3) + d * (sz + 4), "flops": 10 * n}
    if path == "rope":
        n = case["b"] * case["s"] * (case["hq"] + case["hkv"])
        sz = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": n * case["dim"] * sz * 2 + case["b"] * case["s"] * (case["rot"] * 4 + 4),
                "flops": 3 * n * case["rot"]}
    b, s, hq, hkv = case["b"], case["s"], case["hq"], case["hkv"]
    if path == "append":
        back = s + case["page"] - 1
        return {"bytes": b * (s * (hq * HEAD * 4 + hkv * HEAD * 6 + case["rot"] * 4) + back * hkv * HEAD * 6),
                "flops": 6 * b * (s + back) * hkv * HEAD}
    window, sinks = case["window"], case["sinks"]
    pairs = read = 0
    for n in _lengths(case):
        lo = 0
        for p in range(n - s, n):
            w = p + 1 if not window else min(p + 1, window)
            pairs += w + min(sinks, p + 1 - w)
        if window:
            lo = max(0, n - s - window + 1)
        read += n - lo + min(sinks, lo)
    return {"bytes": b * s * hq * (HEAD * 4 + 4) + read * hkv * HEAD * 2, "flops": 4 * hq * HEAD * pairs}


# ------------------------------------------------------------------------- results in 64 bits
def _e4m3_64(x, e):
    """The values that e4m3 numbers of scale 2^e hold for x."""
    f = torch.exp2(e.double())
    return (x / f).clamp(-E4M3, E4M3).to(torch.float8_e4m3fn).double() * f


def _rope64(x, pos, case, inverse=False):
    f, m = _frequencies(case["rot"], case.get("scaling", "none"))
    angle = pos.double()[..., None, None] * f.to(x.device)
    c, s = torch.cos(angle) * m, torch.sin(angle) * m * (-1.0 if inverse else 1.0)
    r, y = case["rot"], x.double().clone()
    one, two = (slice(0, r, 2), slice(1, r, 2)) if case["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
    a, b = x.double()[..., one], x.double()[..., two]
    y[..., one] = a * c - b * s
    y[..., two] = a * s + b * c
    return y


def exact(case, seed):
    r = _raw(case, seed)
    path = case["path"]
    if path.startswith("norm"):
        w = r["w"].double()
        h = r["x"].double()
        if path != "norm_bwd" and r["res"] is not None:
            h = h + r["res"].double()
        size = torch.sqrt(h.square().sum(dim=1, keepdim=True) / case["d"] + EPS)
        n = h / size
        if path == "norm_bwd":
            g = r["dy"].double() * w
            dx = (g - n * (g * n).sum(dim=1, keepdim=True) / case["d"]) / size
            if r["dh"] is not None:
                dx = dx + r["dh"].double()
            return dx, (r["dy"].double() * n).sum(dim=0)
        y = n * w
        if path == "norm_quant":
            b = y.view(y.shape[0], -1, 128)
            sc = b.abs().amax(dim=2, keepdim=True) / E4M3
            if case["pow2"]:
                sc = torch.exp2(torch.ceil(torch.log2(sc)))
            y = ((b / sc).to(torch.float8_e4m3fn).double() * sc).view_as(y)
        return (y, h) if r["res"] is not None else y
    if path == "rope":
        return tuple(_rope64(x, r["pos"], case, case["inverse"]) for x in (r["q"], r["k"]))
    b, s, page, hkv = case["b"], case["s"], case["page"], case["hkv"]
    start = r["start"].tolist()
    if path == "append":
        pos = r["start"][:, None] + torch.arange(s, device=r["q"].device)
        q = _rope64(r["q"], pos, case)
        new = torch.stack((_rope64(r["new"][0], pos, case), r["new"][1].double()))
        back = torch.zeros(2, b, s + page - 1, hkv, HEAD, dtype=torch.float64, device=q.device)
        for i, n in enumerate(start):
            lo = max(0, n - (page - 1)) // page * page
            x = torch.cat((r["kv"][:, i, lo:n].double(), new[:, i]), dim=1)         # tokens lo .. n + s - 1
            for t in range(lo, n + s, page):
                one = x[:, t - lo:t - lo + page]
                old = max(0, min(n - t, page))
                parts = [_exponent(p.abs().amax(dim=(1, 3))) for p in (one[:, :old], one[:, old:]) if p.shape[1]]
                e = torch.stack(parts).amax(dim=0)[:, None, :, None]
                if old:                          # written before the new tokens came
                    one[:, :old] = _e4m3_64(one[:, :old], parts[0][:, None, :, None])
                x[:, t - lo:t - lo + page] = _e4m3_64(one, e)
            want = n - (page - 1)
            back[:, i, max(0, -want):] = x[:, max(0, want) - lo:]
        return q, back[0], back[1]
    o = torch.zeros(b, s, case["hq"], HEAD, dtype=torch.float64, device=r["q"].device)
    lse = torch.zeros(b, case["hq"], s, dtype=torch.float64, device=o.device)
    group = case["hq"] // hkv
    for i, first in enumerate(start):
        n = first + s
        x = r["kv"][:, i, :n].double()
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, (-n) % page)).view(2, -1, page, hkv, HEAD)
        x = _e4m3_64(x, _exponent(x.abs().amax(dim=(2, 4)))[:, :, None, :, None]).view(2, -1, hkv, HEAD)[:, :n]
        j = torch.arange(n, device=o.device)
        for h in range(case["hq"]):
            for at in range(0, s, 2048):
                p = torch.arange(first + at, first + min(at + 2048, s), device=o.device)[:, None]
                sc = r["q"][i, at:at + 2048, h].double() @ x[0, :, h // group].t() / math.sqrt(HEAD)
                hide = j > p
                if case["window"]:
                    hide = hide | ((j <= p - case["window"]) & (j >= case["sinks"]))
                sc = sc.masked_fill(hide, float("-inf"))
                z = torch.logsumexp(sc, dim=1)
                lse[i, h, at:at + 2048] = z
                o[i, at:at + 2048, h] = torch.exp(sc - z[:, None]) @ x[1, :, h // group]
    return o, lse
