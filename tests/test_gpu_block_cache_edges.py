"""Block-scaled cache operators where their arithmetic, argument or layout handling ends.

The helpers and their tolerances are those of test_gpu_block_cache.py.
"""

import numpy as np
import pytest
import torch

import test_gpu_block_cache as base
from test_gpu_alibi import _kernel_names
from test_gpu_block_cache import run_attention

pytestmark = pytest.mark.gpu


def run_prefill(*args, **kw):
    """run_attention on a call that takes the 16-bit copy and the tcgen05 prefill."""
    got = []
    names = _kernel_names(lambda: got.append(run_attention(*args, **kw)))
    assert not names or any("block_copy_kernel" in n for n in names), names
    return got[0]


def dominant_key(nats, v_code, vs_exp=4):
    """Key 2 stands `nats` above all others; its V row holds one code throughout (0: it adds nothing to an output).

    The rest of an output row are the other keys' small probabilities, and the bound
    (relative to sum p |v| / sum p) asks for their own precision.
    """
    def mutate(q, kc, vc, ks, vs, table):
        page = table[0, 0].long()
        q[:, :, 0] = nats / (448 * 2.0 ** -7 * q.shape[-1] ** -0.5)
        raw = kc.view(torch.uint8)
        raw[..., 0] = 0
        raw[page, 2] = 0
        raw[page, 2, :, 0] = 0x7e                        # 448
        ks[page, 0] = 2.0 ** -7
        vc.view(torch.uint8)[page, 2] = v_code
        vs.fill_(2.0 ** vs_exp)                          # outputs stay normal numbers in f16
    return mutate


@pytest.mark.parametrize("v_code", [0, 1])
@pytest.mark.parametrize("nats", [4, 9, 12, 14, 16])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_dominant_key_without_value(dtype, nats, v_code):
    mutate = dominant_key(nats, v_code)
    for hq in (4, 8, 16, 24, 32):                        # every width of the decode kernel
        run_attention([1], [100], hq, 1, 128, 16, 16, dtype, mutate=mutate, q_scale=0.2)
    run_attention([3], [111], 4, 1, 256, 32, 32, dtype, mutate=mutate, q_scale=0.2)
    run_attention([2], [1900], 4, 2, 64, 16, 16, dtype, mutate=mutate, q_scale=0.2, window=100, first=4)
    run_attention([2], [1900], 4, 2, 128, 16, 16, dtype, mutate=mutate, q_scale=0.2, splits=3)


@pytest.mark.parametrize("nats", [4, 9, 12, 14])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_dominant_key_without_value_in_prompt_chunks(d, dtype, nats):
    mutate = dominant_key(nats, 0)
    run_prefill([130, 260], [170, 300], 32, 2, d, 16, 16, dtype, mutate=mutate, q_scale=0.2)
    run_prefill([130, 260], [500, 300], 32, 2, d, 16, 16, dtype, mutate=mutate, q_scale=0.2, window=90, first=4, sinks=True)


@pytest.fixture
def infinite_past_half(monkeypatch):
    """Elements whose exact value rounds to f16's infinity: checked to be that, then taken as exact by run_attention."""
    exact = base.ob.attention
    call = base.flash_attn_with_block_scaled_kvcache

    def checked(q, kc, vc, ks, vs, used, table, **kw):
        out, lse = call(q, kc, vc, ks, vs, used, table, **kw)
        if out.dtype == torch.float16:
            want = exact(base.np_of(q), [base.np_of(kc), base.np_of(vc)], [base.np_of(ks), base.np_of(vs)], used.tolist(),
                         base.np_of(table), base.np_of(kw["cu_seqlens_q"]), q.shape[-1] ** -0.5, kw["causal"],
                         kw["window_size"][0], kw["first_tokens"])[0]
            got = out.double().cpu().numpy()
            past = np.abs(want) >= 65520.0 * (1 + 2.0 ** -9)
            assert np.array_equal(got[past], np.sign(want[past]) * np.inf)
            near = (np.abs(want) >= 65520.0 * (1 - 2.0 ** -9)) & np.isinf(got) & (np.sign(got) == np.sign(want))
            out = FloatOut(out, torch.from_numpy(np.where(past | near, want, got)))
        return out, lse
    monkeypatch.setattr(base, "flash_attn_with_block_scaled_kvcache", checked)


class FloatOut:
    """An output with some elements replaced in 64 bits."""

    def __init__(self, out, values):
        self.dtype, self.shape, self.values = out.dtype, out.shape, values

    def double(self):
        return self.values


@pytest.mark.parametrize("k_exp,v_exp", [(-8, 8), (8, 8), (10, 10), (-22, -22), (12, 40)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scales_beyond_half_precision(dtype, k_exp, v_exp, infinite_past_half):
    """Blocks whose values leave f16's range (an f16 element of 65504 is cached as 256 * 2^8) or its normal numbers."""
    def mutate(q, kc, vc, ks, vs, table):
        for b in range(table.shape[0]):
            page = table[b, 1].long()
            ks[page] = 2.0 ** k_exp
            vs[page] = 2.0 ** v_exp
            if v_exp > 16:                               # of little weight, so that outputs stay finite
                kc.view(torch.uint8)[page] = 0
                kc.view(torch.uint8)[page, :, :, 0] = 0xfe   # -448: a logit of -60 * log(2)
                q[:, :, 0] = 41.6 * q.shape[-1] ** 0.5 / (448 * 2.0 ** k_exp)
                vc.view(torch.uint8)[page] &= 0x81
    q_scale = 2.0 ** -12 if k_exp >= 8 else 1.0
    for ns in ([1, 1], [4, 3]):
        run_attention(ns, [170, 300], 8, 2, 128, 16, 16, dtype, mutate=mutate, q_scale=q_scale)
    for d in (64, 128, 256):
        run_prefill([130, 260], [170, 300], 32, 2, d, 16, 16, dtype, mutate=mutate, q_scale=q_scale)
    run_prefill([130, 260], [500, 300], 32, 2, 128, 32, 32, dtype, mutate=mutate, q_scale=q_scale, window=60, first=40)


@pytest.mark.parametrize("d", [48, 64, 128, 192, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompt_chunks_over_any_scales(dtype, d):
    """Scales that are no powers of two on some KV heads and requests only, blocks of zeros, sinks, first tokens, no causality."""
    def mutate(q, kc, vc, ks, vs, table):
        ks[:, :, 1] *= 1.3                                # one KV head everywhere
        vs[table[1, :2].long(), :, 0] *= 0.77
        for cache, scale in ((kc, ks), (vc, vs)):            # a block of zeros as the append leaves it
            cache.view(torch.uint8)[table[0, 2].long()] = 0
            scale[table[0, 2].long()] = 2.0 ** -100
    args = [130, 260, 0, 9], [171, 300, 40, 9], 32, 4, d, 16, 16, dtype
    run_prefill(*args, mutate=mutate)
    run_prefill(*args, mutate=mutate, sinks=True, window=70, first=20)
    run_prefill(*args, mutate=mutate, sinks=True, causal=False)
    run_prefill([130, 260], [20, 300], 32, 4, d, 16, 16, dtype, mutate=mutate, sinks=True)     # rows that see nothing


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("dtype,d,rot", [(torch.bfloat16, 128, 128), (torch.bfloat16, 128, 64), (torch.float16, 80, 20),
                                         (torch.float32, 128, 128), (torch.bfloat16, 72, 40), (torch.float32, 63, 30)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_writes_query_out(dtype, d, rot, interleaved, in_place, monkeypatch):
    """Queries rotated into a given tensor or in place, by the vector kernels and by the one for any layout."""
    call = base.append_kvcache_block_scaled

    def with_out(*args, query, **kw):
        out = query if in_place else torch.full_like(query, float("nan"))
        assert call(*args, query=query, query_out=out, **kw) is out
        return out
    monkeypatch.setattr(base, "append_kvcache_block_scaled", with_out)
    for ns in ([9, 33, 1], [700, 41, 3]):                # one launch; queries in a launch of their own
        base.run_append(ns, [5, 0, 31], 12, 2, d, 32, 16, dtype, rot=rot, interleaved=interleaved, seed=d)


@pytest.mark.parametrize("V", [1, 2, 33, 257, 1000, 4099, 151936])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_verify_without_residual(V, dtype):
    """Rejected drafts whose q is above p everywhere: the token is drawn from p, whatever the vocabulary's size."""
    def poke(logits, q, tokens, u, noise):
        rows = [0, 1, 2, 4, 7, 8, 9, 10, 11]             # the drafts' rows of requests with 3, 1, 0 and 5 drafts
        q.copy_(torch.softmax(logits[rows].float(), -1) * 1.125)
        u.fill_(0.96875)
    acc = base.run_verify([3, 1, 0, 5], V, dtype, seed=17 + V, poke=poke)
    assert acc.tolist() == [0, 0, 0, 0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("strided", [False, True])
def test_verify_low_temperatures(dtype, strided, monkeypatch):
    """Scores of up to 2^26 at a temperature: only differences to the row's maximum may be scaled by it."""
    call = base.verify_draft_tokens
    if strided:                                          # vocabulary not contiguous
        monkeypatch.setattr(base, "verify_draft_tokens",
                            lambda logits, *args, **kw: call(logits.t().contiguous().t(), *args, **kw))

    def likeliest(logits, q, tokens, u, noise):
        rows = [b + i for b in range(4) for i in range(3 * b, 3 * b + 3)]
        tokens.copy_(logits[rows].float().argmax(-1))
        u.fill_(0.75)
    temps = [1e-6, 1e-5, 1e-4, 1e-3]
    for seed in range(4):
        base.run_verify([3, 3, 3, 3], 1009, dtype, one_hot=True, temps=temps, seed=seed, poke=likeliest)
        base.run_verify([3, 3, 3, 3], 1009, dtype, temps=temps, seed=seed, poke=likeliest)
        base.run_verify([3, 3, 3, 3], 1009, dtype, temps=[1e-2, 3e-2, 1e-1, 30.0], seed=seed)
    base.run_verify([3, 3, 3, 3], 1009, dtype, one_hot=True, temps=[1e-38, 1e-44, 1e30, 1.0], seed=7, poke=likeliest)


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("size", [1e-44, 1e-38, 1e-30, 1.0, 1e30, 2.0 ** 126])
def test_verify_noise_of_any_size(size, strided, monkeypatch):
    """Quotients by the smallest and largest noise that float32 holds, with and without a contiguous vocabulary."""
    call = base.verify_draft_tokens
    if strided:
        monkeypatch.setattr(base, "verify_draft_tokens",
                            lambda logits, *args, **kw: call(logits.t().contiguous().t(), *args, **kw))

    def poke(logits, q, tokens, u, noise):
        g = torch.Generator().manual_seed(5)
        at = torch.randint(1, 3, noise.shape, generator=g)
        noise.copy_(size * at.double())
        logits.copy_(-40.0 - torch.rand(logits.shape, generator=g))
        logits[:, 700] = 1.0                             # probabilities of 0.6 and 0.4 decide
        logits[:, 300] = 0.6
        noise[:, 300] = size * 2
    for one_hot in (False, True):
        base.run_verify([2, 0, 3], 1024, torch.float32, one_hot=one_hot, seed=3, poke=poke)


BIG = 2 ** 31 - 1


@pytest.mark.parametrize("ns,lens", [([1, 1], [300, 129]), ([4, 2], [300, 129]), ([5, 3], [3, 0]), ([130, 260], [500, 300])])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_bounds_of_any_size(dtype, ns, lens):
    """Windows, first tokens and length bounds up to the largest 32-bit number."""
    heads = (32, 2) if max(ns) > 100 else (8, 2)
    if dtype == torch.float32 and max(ns) > 100:
        heads, ns = (2, 1), [40, 60]
    run_attention(ns, lens, *heads, 128, 16, 16, dtype, window=20, first=BIG)
    run_attention(ns, lens, *heads, 128, 16, 16, dtype, window=BIG, first=3)
    run_attention(ns, lens, *heads, 128, 16, 16, dtype, window=BIG - 1, first=BIG, max_k=BIG)
    g = torch.Generator().manual_seed(1)
    kc, vc, ks, vs, table = base.make_cache(g, lens, 16, 16, heads[1], 128)
    q = torch.randn(sum(ns), heads[0], 128, generator=g).to(dtype).cuda()
    used, cu = torch.tensor(lens, dtype=torch.int32).cuda(), base.offsets(ns)
    call = base.flash_attn_with_block_scaled_kvcache
    want = call(q, kc, vc, ks, vs, used, table, cu_seqlens_q=cu, max_seqlen_q=sum(ns), max_seqlen_k=table.shape[1] * 16)
    got = call(q, kc, vc, ks, vs, used, table, cu_seqlens_q=cu, max_seqlen_q=BIG, max_seqlen_k=BIG)
    assert torch.equal(got, want)


def test_append_refuses_positions_without_axes():
    g = torch.Generator().manual_seed(1)
    kc, vc, ks, vs, table = base.make_cache(g, [64, 64], 16, 16, 2, 128)
    k = torch.randn(2, 1, 2, 128, generator=g).to(torch.bfloat16).cuda()
    used = torch.tensor([3, 9], dtype=torch.int32).cuda()
    cos = torch.ones(64, 64).cuda()
    with pytest.raises(ValueError, match="axis"):
        base.append_kvcache_block_scaled(k, k, kc, vc, ks, vs, used, table, rotary_cos=cos, rotary_sin=cos,
                                         positions=torch.zeros(0, 2, dtype=torch.int32).cuda())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_bounds_of_any_size(dtype, monkeypatch):
    """Any upper bound of new tokens; requests whose length lies behind their table row append nothing."""
    call = base.append_kvcache_block_scaled
    monkeypatch.setattr(base, "append_kvcache_block_scaled", lambda *args, **kw: call(*args, **dict(kw, max_seqlen=BIG)))
    base.run_append([1, 5, 0, 37], [0, 15, 3, 130], 6, 2, 128, 64, 32, dtype)
    base.run_append([1, 1], [63, 64], 6, 2, 128, 64, 64, dtype)
    g = torch.Generator().manual_seed(1)
    kc, vc, ks, vs, table = base.make_cache(g, [64, 64, 64], 16, 16, 2, 128)
    x = torch.randn(90, 2, 128, generator=g).to(dtype).cuda()
    lens = [BIG - 20, table.shape[1] * 16, -5]
    before = [base.np_of(t).copy() for t in (kc, vc, ks, vs)]
    call(x, x, kc, vc, ks, vs, torch.tensor(lens, dtype=torch.int32).cuda(), table, cu_seqlens=base.offsets([15, 40, 35]),
         max_seqlen=BIG)
    for t, want in zip((kc, vc, ks, vs), before):
        assert np.array_equal(base.np_of(t), want)


@pytest.mark.parametrize("ns", [[1, 1], [4, 3], [130, 260]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_nan_rows_stay_nan(dtype, ns):
    """A NaN in a query or in a visible key makes exactly the rows that see it NaN, whatever kernel takes the call."""
    heads, lens, d, at = (32, 4), [500, 300], 128, 299
    if dtype == torch.float32 and max(ns) > 100:
        heads, ns = (4, 2), [60, 40]
    g = torch.Generator().manual_seed(3)
    kc, vc, ks, vs, table = base.make_cache(g, lens, 16, 16, heads[1], d)
    T = sum(ns)
    q = torch.randn(T, heads[0], d, generator=g).to(dtype).cuda()
    used, cu = torch.tensor(lens, dtype=torch.int32).cuda(), base.offsets(ns)
    call = lambda: base.flash_attn_with_block_scaled_kvcache(
        q, kc, vc, ks, vs, used, table, cu_seqlens_q=cu, max_seqlen_q=max(ns), max_seqlen_k=max(lens), return_softmax_lse=True)
    want, want_lse = call()
    q[0, 1, 7] = float("nan")
    kc.view(torch.uint8)[table[1, at // 16].long(), at % 16, 0, 5] = 0x7f     # the last key of request 1, KV head 0
    out, lse = call()
    nan = torch.zeros(T, heads[0], dtype=torch.bool, device="cuda")
    nan[0, 1] = True
    nan[-1, :heads[0] // heads[1]] = True                                      # only the last query sees it
    assert torch.equal(torch.isnan(out), nan[..., None].expand_as(out))
    assert torch.equal(torch.isnan(lse), nan.T)
    assert torch.equal(out[~nan], want[~nan]) and torch.equal(lse.T[~nan], want_lse.T[~nan])


@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-25, 3.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_softmax_scales(dtype, scale):
    """Scales that are zero, negative, tiny or large, for single tokens and prompt chunks."""
    for ns, q_scale in (([1, 3], 1.0), ([130, 260], 1.0)):
        g = torch.Generator().manual_seed(9)
        lens = [300, 270]
        kc, vc, ks, vs, table = base.make_cache(g, lens, 16, 16, 2, 128)
        q = (torch.randn(sum(ns), 16, 128, generator=g) * q_scale).to(dtype).cuda()
        used, cu = torch.tensor(lens, dtype=torch.int32).cuda(), base.offsets(ns)
        out, lse = base.flash_attn_with_block_scaled_kvcache(
            q, kc, vc, ks, vs, used, table, cu_seqlens_q=cu, max_seqlen_q=max(ns), max_seqlen_k=max(lens),
            softmax_scale=scale, return_softmax_lse=True)
        want, want_lse, spread = base.ob.attention(
            base.np_of(q), [base.np_of(kc), base.np_of(vc)], [base.np_of(ks), base.np_of(vs)], lens, base.np_of(table),
            base.np_of(cu), float(np.float32(scale)))
        err = np.abs(lse.double().cpu().numpy() - want_lse)
        assert (err <= 2e-5 + 2e-6 * np.abs(want_lse)).all(), err.max()
        err = np.abs(out.double().cpu().numpy() - want)
        assert (err <= base.EPS[dtype] * (np.abs(want) + spread) + 2e-5 * spread + 1e-7).all(), err.max()


# Kernels and routes that sizes of real use reach, at small ones.
@pytest.mark.parametrize("splits", [0, 2, 5, 60])
@pytest.mark.parametrize("d", [128, 256])
def test_sinks_over_joined_pieces(d, splits):
    run_attention([1, 1, 0, 1], [2100, 700, 5, 0], 8, 2, d, 16, 16, torch.bfloat16, sinks=True, splits=splits)
    run_attention([3, 1], [1500, 900], 8, 2, d, 32, 16, torch.float16, sinks=True, splits=splits, window=600, first=130)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompt_chunks_in_several_passes(dtype, monkeypatch):
    """A block table of 640000 tokens a request: the copies of two requests do not go into one pass."""
    make = base.make_cache

    def wide_table(*args, **kw):
        *cache, table = make(*args, **kw)
        return *cache, torch.cat([table, torch.full((table.shape[0], 40000), -1, dtype=torch.int32, device="cuda")], dim=1)
    monkeypatch.setattr(base, "make_cache", wide_table)
    run_prefill([130, 260, 17], [171, 300, 900], 32, 2, 128, 16, 16, dtype, max_k=640000, sinks=True)
    run_prefill([130, 260, 17], [171, 300, 900], 32, 2, 128, 16, 16, dtype, max_k=640000, window=100, first=4,
                mutate=lambda q, kc, vc, ks, vs, table: ks[:, :, 1].mul_(1.3))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_append_wide_heads_and_blocks(dtype):
    """Units of 16 warps: blocks of 128 tokens with head dims above 128."""
    for d, page in ((256, 128), (192, 256), (144, 128)):
        base.run_append([200, 1, 131, 64], [0, 127, 70, 130], 4, 2, d, page, 128, dtype, seed=d)
        base.run_append([17], [250], 4, 2, d, page, 128, dtype, seed=d, axes=3, interleaved=True)


def test_verify_many_drafts():
    """More drafts than a request's numbers in shared memory; all accepted, and rejected behind them."""
    def accept(until):
        def poke(logits, q, tokens, u, noise):
            rows = list(range(100)) + list(range(101, 104))
            tokens.copy_(logits[rows].argmax(-1))
            u.fill_(0.5)
            u[until] = 0.99999
            logits[rows[until], 3] = logits[rows[until]].max()
            logits[rows[until], 4] = logits[rows[until]].max()
        return poke
    for until in (0, 63, 64, 65, 99):
        for temps in ([1e-3, 1.0], [0.0, 0.0]):
            base.run_verify([100, 3], 61, torch.float32, one_hot=True, temps=temps, seed=2, poke=accept(until))


def test_verify_more_rows_than_a_grid():
    g = torch.Generator().manual_seed(4)
    B, V = 40000, 3
    logits = torch.randn(2 * B, V, generator=g).cuda() * 3
    tokens = torch.randint(0, V, (B,), generator=g).cuda()
    cu = torch.arange(B + 1, dtype=torch.int32).cuda()
    u, noise = torch.rand(B, generator=g).cuda(), torch.empty(B, V).exponential_(generator=g).clamp_(min=1e-20).cuda()
    got = base.verify_draft_tokens(logits, tokens, cu, u, noise, max_draft=1)
    want, acc, _ = base.ob.verify(base.np_of(logits), base.np_of(tokens), base.np_of(cu), base.np_of(u), base.np_of(noise),
                                  None, None, 1)
    # Of 80000 random decisions about 80000 * 1e-6 may lie within float32's rounding.
    assert (got[0].cpu().numpy() != want).any(1).sum() + (got[1].cpu().numpy() != acc).sum() <= 3


def test_append_refuses_queries_without_heads():
    g = torch.Generator().manual_seed(1)
    kc, vc, ks, vs, table = base.make_cache(g, [64, 64], 16, 16, 2, 128)
    used = torch.tensor([3, 9], dtype=torch.int32).cuda()
    for new in (1, 600):
        k = torch.randn(2, new, 2, 128, generator=g).to(torch.bfloat16).cuda()
        with pytest.raises(ValueError, match="heads"):
            base.append_kvcache_block_scaled(k, k, kc, vc, ks, vs, used, table, query=k[:, :, :0])


@pytest.mark.parametrize("dtype,odd", [(torch.bfloat16, False), (torch.float16, True)])
def test_prompt_chunks_in_a_cuda_graph(dtype, odd):
    """A captured prompt chunk replayed over another cache content, with scales that both launches take: equal to eager calls."""
    g = torch.Generator().manual_seed(6)
    lens, ns = [300, 280], [130, 260]
    kc, vc, ks, vs, table = base.make_cache(g, lens, 16, 16, 2, 128)
    used, cu = torch.tensor(lens, dtype=torch.int32).cuda(), base.offsets(ns)
    q = torch.randn(sum(ns), 32, 128, generator=g).to(dtype).cuda()

    def step():
        return base.flash_attn_with_block_scaled_kvcache(q, kc, vc, ks, vs, used, table, cu_seqlens_q=cu, max_seqlen_q=260,
                                                         max_seqlen_k=300, return_softmax_lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (1, 2):
        h = torch.Generator().manual_seed(seed)
        q.copy_(torch.randn(q.shape, generator=h).to(dtype))
        if odd:
            ks[:, :, seed - 1] *= 1.7
        graph.replay()
        got = [t.clone() for t in captured]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


@pytest.fixture
def poisoned_workspaces(monkeypatch):
    """Workspaces and outputs begin as NaN in every type."""
    new_empty = torch.Tensor.new_empty

    def poisoned(self, *args, **kw):
        t = new_empty(self, *args, **kw)
        if t.numel():
            t.view(torch.uint8).fill_(0xff)
        return t
    monkeypatch.setattr(torch.Tensor, "new_empty", poisoned)


@pytest.mark.parametrize("hk,d", [(1, 48), (2, 48), (3, 48), (3, 128), (5, 80), (3, 208)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_nothing_left_in_workspaces_is_read(dtype, hk, d, poisoned_workspaces):
    """Ends of requests inside a tile, heads of both scale forms side by side, pieces and merges, over poisoned memory."""
    def mutate(q, kc, vc, ks, vs, table):
        ks[:, :, 0] *= 1.3
    for mutation in (None, mutate):
        run_prefill([130, 260], [171, 300], 32 // hk * hk, hk, d, 16, 16, dtype, mutate=mutation)
        run_prefill([260, 130], [900, 131], 32 // hk * hk, hk, d, 16, 16, dtype, mutate=mutation, window=200, first=130)
    for splits in (0, 1, 3, 40):
        run_attention([1, 0, 1, 2], [171, 9, 1300, 5], 2 * hk, hk, d, 16, 16, dtype, mutate=mutate, splits=splits)
        run_attention([1, 0, 1, 2], [171, 9, 1300, 5], 2 * hk, hk, d, 16, 16, dtype, splits=splits, window=300, first=5)


def test_verification_reads_nothing_left_in_its_workspace(poisoned_workspaces):
    for V in (1, 1000, 4097, 151936):
        base.run_verify([3, 0, 1, 5, 2], V, torch.bfloat16, temps=[0.7, 1.0, 0.0, 1.3, 0.0], seed=11 + V)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_behind_any_scales_and_positions(dtype, monkeypatch):
    """Older scales that are no powers of two; positions in front of and behind the tables."""
    make = base.make_cache

    def scaled(*args, **kw):
        kc, vc, ks, vs, table = make(*args, **kw)
        return kc, vc, ks * 1.375, vs * 0.8125, table
    monkeypatch.setattr(base, "make_cache", scaled)
    base.run_append([9, 33, 1, 130], [5, 10, 31, 17], 6, 2, 128, 32, 16, dtype, scale=8.0)
    base.run_append([9, 33, 1, 130], [5, 10, 31, 17], 6, 2, 128, 64, 64, dtype, scale=0.1)
    call = base.append_kvcache_block_scaled

    def shifted(*args, positions, **kw):
        assert (positions < 0).any() and (positions >= kw["rotary_cos"].shape[0]).any()
        return call(*args, positions=positions, **kw)
    monkeypatch.setattr(base, "append_kvcache_block_scaled", shifted)
    randint = torch.randint
    monkeypatch.setattr(torch, "randint", lambda lo, hi, *a, **kw: randint(lo - 50 if kw.get("dtype") == torch.int32 else lo,
                                                                           hi + 50 if kw.get("dtype") == torch.int32 else hi, *a, **kw))
    base.run_append([9, 33, 90], [5, 10, 17], 6, 2, 128, 32, 16, dtype)
    base.run_append([9, 33, 90], [5, 10, 17], 6, 2, 128, 32, 16, dtype, axes=3)


def strided_copy(x, dims):
    """x's values with other strides: dimensions stored in the order `dims`, two elements apart."""
    out = torch.zeros(*[x.shape[i] for i in dims], 2, dtype=x.dtype, device=x.device)[..., 1]
    out = out.permute(*[dims.index(i) for i in range(x.ndim)])
    return out.copy_(x)


def heads_first(cache):
    """A cache stored heads before tokens."""
    raw = cache.view(torch.uint8).permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    return raw.view(torch.float8_e4m3fn)


@pytest.mark.parametrize("ns", [[1, 1], [5, 3], [130, 260]])
def test_strided_scales_tables_and_lengths(ns):
    """Every small tensor strided, K and V caches of different layouts: equal to the contiguous call."""
    g = torch.Generator().manual_seed(2)
    lens = [500, 300]
    kc, vc, ks, vs, table = base.make_cache(g, lens, 32, 16, 2, 128)
    q = torch.randn(sum(ns), 16, 128, generator=g).to(torch.bfloat16).cuda()
    k, v = torch.randn(2, sum(ns), 2, 128, generator=g).to(torch.bfloat16).cuda()
    starts = torch.tensor(lens, dtype=torch.int32).cuda() - torch.tensor(ns, dtype=torch.int32).cuda()
    used, cu = torch.tensor(lens, dtype=torch.int32).cuda(), base.offsets(ns)
    angle = torch.rand(600, 64, generator=g).cuda()
    cos, sin, pos = angle.cos(), angle.sin(), torch.randint(0, 600, (sum(ns),), generator=g, dtype=torch.int32).cuda()
    aux = torch.randn(16, generator=g).cuda()

    def step(kc, vc, ks, vs, table, starts, used, cu, cos, sin, pos, aux):
        r = base.append_kvcache_block_scaled(k, v, kc, vc, ks, vs, starts, table, cu_seqlens=cu, max_seqlen=max(ns), query=q,
                                             rotary_cos=cos, rotary_sin=sin, positions=pos)
        return r, *base.flash_attn_with_block_scaled_kvcache(r, kc, vc, ks, vs, used, table, cu_seqlens_q=cu, max_seqlen_q=max(ns),
                                                             max_seqlen_k=500, s_aux=aux, return_softmax_lse=True), kc, vc, ks, vs
    contiguous = (kc.clone(), vc.clone(), ks.clone(), vs.clone(), table, starts, used, cu, cos, sin, pos, aux)
    strided = (kc, heads_first(vc), strided_copy(ks, (2, 0, 1)), strided_copy(vs, (1, 2, 0)), strided_copy(table, (1, 0)),
               *[strided_copy(t, (0,)) for t in (starts, used, cu)], strided_copy(cos, (0, 1)), strided_copy(sin, (1, 0)),
               strided_copy(pos, (0,)), strided_copy(aux, (0,)))
    for a, b in zip(step(*contiguous), step(*strided)):
        if a.dtype == torch.float8_e4m3fn:
            a, b = a.view(torch.uint8), b.view(torch.uint8)
        assert torch.equal(a, b)


@pytest.mark.parametrize("ns", [[1, 1], [130, 260]])
def test_offsets_past_32_bits(ns):
    """Pages more than 2^31 bytes into the cache: equal to the same pages in a small one."""
    g = torch.Generator().manual_seed(2)
    lens, page, hk, d = [500, 300], 128, 8, 128
    small = base.make_cache(g, lens, page, 128, hk, d)
    pages = 2 ** 31 // (page * hk * d) + 20
    far = pages - small[0].shape[0]
    big = [torch.zeros(pages, page, hk, d, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)]
    big += [torch.ones(pages, 1, hk, device="cuda") for _ in range(2)]
    for x, y in zip(big, small):
        x.view(torch.uint8)[far:].copy_(y.view(torch.uint8))
    table = torch.where(small[4] >= 0, small[4] + far, -1)
    q = torch.randn(sum(ns), 32, d, generator=g).to(torch.bfloat16).cuda()
    k, v = torch.randn(2, sum(ns), hk, d, generator=g).to(torch.bfloat16).cuda()
    used, cu = torch.tensor(lens, dtype=torch.int32).cuda(), base.offsets(ns)
    starts = used - torch.tensor(ns, dtype=torch.int32).cuda()
    got = []
    for cache, t in ((big, table), (small[:4], small[4])):
        base.append_kvcache_block_scaled(k, v, *cache, starts, t, cu_seqlens=cu, max_seqlen=max(ns))
        got.append(base.flash_attn_with_block_scaled_kvcache(q, *cache, used, t, cu_seqlens_q=cu, max_seqlen_q=max(ns),
                                                             max_seqlen_k=500, return_softmax_lse=True))
        got[-1] += tuple(x.view(torch.uint8)[far if cache is big else 0:] for x in cache)
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_verify_offsets_past_32_bits():
    g = torch.Generator().manual_seed(3)
    V, stride = 1024, 3 * 2 ** 29
    want = torch.randn(4, V, generator=g).to(torch.bfloat16).cuda()
    logits = torch.empty(3 * stride + V, dtype=torch.bfloat16, device="cuda").as_strided((4, V), (stride, 1))
    logits.copy_(want)
    tokens = torch.randint(0, V, (2,), generator=g).cuda()
    u, noise = torch.rand(2, generator=g).cuda() * 1e-4, torch.rand(2, V, generator=g).cuda() + 0.01
    calls = [base.verify_draft_tokens(x, tokens, base.offsets([2, 0]), u, noise, max_draft=2) for x in (logits, want)]
    assert all(torch.equal(a, b) for a, b in zip(*calls))
