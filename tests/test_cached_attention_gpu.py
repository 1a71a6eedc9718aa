"""The attention block over the 8-bit cache, prompts and single tokens, against the block in fp32; and the short call
path of its operators against the general one."""
import pytest
import torch

pytestmark = pytest.mark.gpu

# Relative error in the 2-norm of a product of two e4m3 operands, 2^-4 / sqrt(3) each; keys and values in e4m3 once
# more; the block's result carries the values' and, through the weights, part of the others'.
REL = 3 * 2.0 ** -4 / 3 ** 0.5


@pytest.mark.parametrize("window,sinks,rope", [(0, 0, None), (40, 3, dict(rot=64, interleaved=True))])
def test_block_matches_fp32_for_prompts_and_tokens(native_lib, window, sinks, rope):
    from commbench_b200.models.cached_attention import CachedAttention

    B, S, hidden, steps = 2, 150, 512, 5
    blk = CachedAttention(hidden, heads=8, kv_heads=2, num_pages=16, max_positions=256, page=32, window=window,
                          sinks=sinks, rope=rope)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(B, S + steps, hidden, device="cuda", generator=g).bfloat16()
    want = blk.reference(x)
    pages = torch.randperm(16, device="cuda", generator=g).int()[:10].view(B, 5).contiguous()
    start = torch.zeros(B, dtype=torch.int32, device="cuda")
    # the prompt in two chunks, the second of no round length, then token by token
    got, at = [], 0
    for n in (100, 50) + (1,) * steps:
        y, h = blk.forward(x[:, at:at + n].contiguous(), pages, start)
        assert torch.equal(h, x[:, at:at + n])
        got.append(y)
        start += n
        at += n
    got = torch.cat(got, dim=1).float()
    for rows in (got[:, :S], got[:, S:]), (want[:, :S], want[:, S:]):
        assert all(torch.isfinite(r).all() for r in rows)
    assert ((got - want).norm() / want.norm()).item() < REL
    assert ((got[:, S:] - want[:, S:]).norm() / want[:, S:].norm()).item() < REL


def test_block_with_residual_and_counts(native_lib):
    from commbench_b200.models.cached_attention import CachedAttention

    blk = CachedAttention(256, heads=4, kv_heads=4, num_pages=8, max_positions=128, page=64)
    g = torch.Generator(device="cuda").manual_seed(2)
    x, r = (torch.randn(2, 20, 256, device="cuda", generator=g).bfloat16() for _ in range(2))
    pages = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2)
    start = torch.zeros(2, dtype=torch.int32, device="cuda")
    count = torch.tensor([20, 13], dtype=torch.int32, device="cuda")
    y, h = blk.forward(x, pages, start, count=count, residual=r)
    assert torch.equal(h, (x.float() + r.float()).bfloat16())
    want = blk.reference((x.float() + r.float()))
    assert (y[1, 13:] == 0).all()
    assert ((y[0].float() - want[0]).norm() / want[0].norm()).item() < REL
    assert ((y[1, :13].float() - want[1, :13]).norm() / want[1, :13].norm()).item() < REL


def test_short_and_general_call_path_agree(native_lib, monkeypatch):
    from commbench_b200 import _native as N
    from commbench_b200.ops.kvcache import KVCache8
    from commbench_b200.ops.norm import rms_norm, rms_norm_backward, rms_norm_quant
    from commbench_b200.ops.rope import RopeTable, rope

    g = torch.Generator(device="cuda").manual_seed(3)
    x, r = (torch.randn(37, 512, device="cuda", generator=g).bfloat16() for _ in range(2))
    w = torch.randn(512, device="cuda", generator=g).bfloat16()
    qkv = torch.randn(3, 70, 12, 128, device="cuda", generator=g).bfloat16()
    q, k, v = qkv.split((8, 2, 2), dim=2)
    pages = torch.randperm(12, device="cuda", generator=g).int().view(3, 4)
    start = torch.zeros(3, dtype=torch.int32, device="cuda")
    count = torch.tensor([70, 5, 33], dtype=torch.int32, device="cuda")
    table, pos = RopeTable(96, 200, interleaved=True), torch.arange(70, device="cuda")

    def everything():
        cache = KVCache8(12, 2, page=32)
        out = [*rms_norm(x, w, residual=r), rms_norm(x, w), *rms_norm_quant(x, w, pow2=True)[:3],
               *rms_norm_quant(x, w, residual=r), *rms_norm_backward(x, r, w, dh=x), *rms_norm_backward(x, r, w),
               rope(q, pos, table), *rope((q, k), pos, table, inverse=True)]
        out.append(cache.append(k, v, pages, start, count=count, rope=table, q=q))
        assert cache.append(k, v, pages, start, count=count) is None
        out += cache.read(pages, start - 3, 40, length=count)
        out += cache.read(pages, None, 70)
        out += cache.attend(q, pages, start, count=count)
        out += cache.attend(q[:, :1], pages, count - 1, window=20, sinks=2, scale=0.1, max_len=100)
        return out

    class Refuses:
        def __getattr__(self, name):
            return lambda *args: None

    fast = N.fast()
    calls = []

    class Counts:
        def __getattr__(self, name):
            f = getattr(fast, name)

            def call(*args):
                res = f(*args)
                calls.append((name, res is not None))
                return res
            return call

    monkeypatch.setattr(N, "fast", lambda: Counts())
    a = everything()
    assert all(taken for _, taken in calls), calls
    monkeypatch.setattr(N, "fast", lambda: Refuses())
    b = everything()
    for i, (s, t) in enumerate(zip(a, b, strict=True)):
        assert s.dtype == t.dtype and s.shape == t.shape, i
        assert torch.equal(s.view(torch.uint8) if s.dtype == torch.float8_e4m3fn else s,
                           t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t), i
