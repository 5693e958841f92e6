"""Attention of a served layer: the three operators against plain implementations in 64 bits.

Bounds, with u the unit roundoff of the 16-bit type (2^-8 bf16, 2^-11 fp16):
  scores   a sum of D products of 16-bit numbers in fp32, scaled: off by at most d = scale (D + 8) 2^-24 max sum |q k| + 2^-20
           (the last term covers exp2 and the running sums)
  weights  exp of that, rounded once to 16 bits: relative error u + 2 d; in fp16 also 2^-25 absolute, per key
  output   |error| <= u |out| + (u + 2 d) sum w |v| [+ keys 2^-25 max |v| in fp16], the last rounding and the weights'
  lse      2 d + 2^-20 (1 + |lse|)
Rotation: (a cos - b sin) takes three fp32 roundings, 2^-22 (|a| + |b|), and the rounding of the result.
"""
import math

import pytest
import torch

import mslk_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F8 = torch.float8_e4m3fn
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def offsets(lengths):
    return torch.tensor([0] + list(lengths), dtype=torch.int32).cumsum(0).to(torch.int32)


def attention(q, k, v, scale, visible):
    """q [n, hq, d], k, v [t, hkv, d] in any float type on the CPU, visible [n, t] -> out, lse, bound of out, bound of lse (64 bits)."""
    n, hq, d = q.shape
    t, hkv, _ = k.shape
    dtype = q.dtype
    q, k, v = q.double(), k.double(), v.double()
    k, v = (x.repeat_interleave(hq // hkv, 1) for x in (k, v))
    s = torch.einsum("nhd,thd->hnt", q, k) * scale
    s = s.masked_fill(~visible, -math.inf)
    lse = torch.logsumexp(s, -1)
    w = torch.exp(s - lse[..., None].masked_fill(lse[..., None] == -math.inf, 0.0))
    out = torch.einsum("hnt,thd->nhd", w, v)
    u = ROUND[dtype]
    if t:
        size = torch.einsum("nhd,thd->hnt", q.abs(), k.abs()).amax(-1).T[..., None]   # [n, hq, 1]
    else:
        size = torch.zeros(n, hq, 1, dtype=torch.float64)
    delta = scale * (d + 8) * 2.0 ** -24 * size + 2.0 ** -20
    bound = u * out.abs() + (u + 2 * delta) * torch.einsum("hnt,thd->nhd", w, v.abs())
    if dtype == torch.float16:
        bound += 2.0 ** -25 * (1 + visible.sum(-1)[:, None, None] * (v.abs().max() if t else 0.0))
    bound += 1e-38
    lse = lse.T
    return out, lse, bound, (2 * delta[..., 0] + 2.0 ** -20 * (1 + lse.abs()))


def near(got, want, bound, what=""):
    got = got.double().cpu()
    assert got.shape == want.shape
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    assert torch.equal(got[~finite & ~torch.isnan(want)], want[~finite & ~torch.isnan(want)]), f"{what}: infinities differ"
    over = ((got - want).abs() - bound)[finite]
    assert over.numel() == 0 or over.max() <= 0, f"{what}: {int((over > 0).sum())} of {over.numel()} beyond the bound, worst by {over.max():.3e}"


def heads(g, tokens, n, d, dtype):
    return torch.randn(tokens, n, d, generator=g).to(dtype)


# ---------------------------------------------------------------------------------------------------------------------
# prompts
# ---------------------------------------------------------------------------------------------------------------------
def causal_mask(n, t):
    return torch.arange(t)[None] <= torch.arange(n)[:, None] + (t - n)


def check_prompt(q, k, v, lens, lens_k=None, causal=True, scale=None, got=None):
    """q, k, v on the CPU; `got`: outputs of a call made by the test."""
    d = q.shape[-1]
    if got is None:
        got = mslk_amd.attention_prompt(q.to(DEV), k.to(DEV), v.to(DEV), offsets(lens).to(DEV),
                                        None if lens_k is None else offsets(lens_k).to(DEV), causal=causal, scale=scale, return_lse=True)
    scale = d ** -0.5 if scale is None else scale
    at_q = at_k = 0
    for b, (n, t) in enumerate(zip(lens, lens if lens_k is None else lens_k)):
        visible = causal_mask(n, t) if causal else torch.ones(n, t, dtype=torch.bool)
        out, lse, bound, lse_bound = attention(q[at_q:at_q + n], k[at_k:at_k + t], v[at_k:at_k + t], scale, visible)
        near(got[0][at_q:at_q + n], out, bound, f"sequence {b}")
        near(got[1][at_q:at_q + n], lse, lse_bound, f"lse of sequence {b}")
        at_q, at_k = at_q + n, at_k + t
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [8, 64, 72, 80, 96, 112, 128, 136, 192, 200, 256])
def test_prompt_head_dimensions(d, dtype):
    g = torch.Generator().manual_seed(d)
    lens = [1, 130, 65]
    q, k, v = heads(g, sum(lens), 4, d, dtype), heads(g, sum(lens), 2, d, dtype), heads(g, sum(lens), 2, d, dtype)
    check_prompt(q, k, v, lens)


@pytest.mark.parametrize("lens", [[1], [2], [31], [32], [33], [63], [64], [65], [127], [128], [129], [255, 257], [0, 5, 0, 0, 200, 0],
                                  [1] * 70, [3, 1, 4, 1, 5, 9, 2, 6] * 17, [700]])
def test_prompt_lengths(lens):
    g = torch.Generator().manual_seed(sum(lens))
    q, k, v = heads(g, sum(lens), 2, 128, torch.bfloat16), heads(g, sum(lens), 1, 128, torch.bfloat16), heads(g, sum(lens), 1, 128, torch.bfloat16)
    for causal in (True, False):
        check_prompt(q, k, v, lens, causal=causal)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (5, 5), (8, 8), (16, 8), (24, 8), (40, 8), (7, 1), (48, 16)])
def test_prompt_head_layouts(hq, hkv):
    g = torch.Generator().manual_seed(hq)
    lens = [150, 20]
    q, k, v = heads(g, 170, hq, 64, torch.bfloat16), heads(g, 170, hkv, 64, torch.bfloat16), heads(g, 170, hkv, 64, torch.bfloat16)
    check_prompt(q, k, v, lens)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,lens_k", [([5, 100, 1], [70, 300, 64]), ([100, 3, 130], [40, 0, 1]), ([4, 4], [0, 0]), ([0, 300], [10, 301]), ([1], [1000])])
def test_prompt_other_key_lengths(lens, lens_k, causal):
    """Continued prompts; more queries than keys: the first ones see nothing; no keys at all."""
    g = torch.Generator().manual_seed(3)
    q = heads(g, sum(lens), 4, 64, torch.float16)
    k, v = heads(g, sum(lens_k), 2, 64, torch.float16), heads(g, sum(lens_k), 2, 64, torch.float16)
    out, lse = check_prompt(q, k, v, lens, lens_k, causal)
    if causal and lens[0] > lens_k[0]:
        unseeing = lens[0] - lens_k[0]
        assert (out[:unseeing] == 0).all() and (lse[:unseeing] == -math.inf).all()


def test_prompt_tokens_of_no_sequence_give_zeros():
    g = torch.Generator().manual_seed(4)
    q, k, v = (heads(g, 400, 2, 64, torch.bfloat16) for _ in range(3))
    k[300:], v[300:], q[300:] = math.nan, math.nan, math.nan   # padding of a fixed-size batch
    k[:7], v[:7] = math.inf, math.nan
    cu = torch.tensor([7, 100, 100, 300], dtype=torch.int32)
    out, lse = mslk_amd.attention_prompt(*(x.to(DEV) for x in (q, k, v)), cu.to(DEV), return_lse=True)
    for part in (slice(0, 7), slice(300, 400)):
        assert (out[part] == 0).all() and (lse[part] == -math.inf).all()
    check_prompt(q[7:300], k[7:300], v[7:300], [93, 0, 200], got=(out[7:300], lse[7:300]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompt_wild_values_stay_behind_the_mask(dtype):
    """A NaN or an infinity in a key or a value touches the queries that see it and no others."""
    g = torch.Generator().manual_seed(5)
    lens = [200, 90]
    base = [heads(g, 290, 2, 128, dtype) for _ in range(3)]
    for where in (0, 1, 40, 63, 64, 100, 127, 130, 199):
        for bad in (math.nan, math.inf, -math.inf):
            q, k, v = (x.clone() for x in base)
            v[where, 1, 5] = bad
            got = mslk_amd.attention_prompt(*(x.to(DEV) for x in (q, k, v)), offsets(lens).to(DEV), return_lse=True)
            clean = check_prompt(*base, lens)
            out = got[0].double().cpu()
            seen = torch.zeros_like(out, dtype=torch.bool)
            seen[where:200, 1, 5] = True
            assert torch.equal(out[~seen], clean[0].double().cpu()[~seen]), (where, bad)
            if math.isnan(bad):
                assert torch.isnan(out[seen]).all()
            else:
                assert (out[seen] == bad).all()
            k[where, 0, 3] = math.nan
            out = mslk_amd.attention_prompt(*(x.to(DEV) for x in (q, k, base[2])), offsets(lens).to(DEV)).double().cpu()
            assert torch.isnan(out[where:200, 0]).all() and torch.equal(out[:where], clean[0].double().cpu()[:where])
            assert torch.equal(out[200:], clean[0].double().cpu()[200:])


def test_prompt_scores_far_apart():
    """Large scores: the running maximum moves by hundreds between tiles, up and down."""
    g = torch.Generator().manual_seed(6)
    q, k, v = (heads(g, 500, 2, 64, torch.bfloat16) for _ in range(3))
    k[100:110] *= 60
    k[300] *= 200
    k[420:] *= 0.01
    check_prompt(q, k, v, [500])
    check_prompt(q, k, v, [500], scale=3.0)
    check_prompt(q, k, v, [500], scale=1e-4, causal=False)


@pytest.mark.parametrize("scale", [1e-44, 1e-38, 1.5e-38, 1e-30, 1e30, 2e38])
def test_scales_at_the_ends_of_their_range(scale):
    """Tiny: every key weighs the same, in however many tiles.  Huge: scores of 0 and of minus the scale, so that the first
    kind alone counts; lse = log of their number."""
    g = torch.Generator().manual_seed(10)
    n, d = 330, 64
    q, k, v = torch.zeros(n, 2, d).bfloat16(), torch.zeros(n, 2, d).bfloat16(), heads(g, n, 2, d, torch.bfloat16)
    q[:, :, 0] = 1
    counts = torch.arange(n) % 3 == 0
    k[~counts, :, 0] = -1
    weighs = counts if scale > 1 else torch.ones(n, dtype=torch.bool)
    out, lse, bound, lse_bound = attention(q, torch.zeros_like(k), v, 1.0, causal_mask(n, n) & weighs)
    got = mslk_amd.attention_prompt(*(x.to(DEV) for x in (q, k, v)), offsets([n]).to(DEV), scale=scale, return_lse=True)
    near(got[0], out, bound)
    near(got[1], lse, lse_bound)
    for length in (n, 5):
        cache = Cache(g, [length], 2, d, 16, torch.bfloat16, extra=100, rows=[[k[:length]], [v[:length]]])
        got = mslk_amd.attention_decode(q[:1].to(DEV), *cache.on_gpu(), scale=scale, return_lse=True)
        near(got[0], out[length - 1:length], bound[length - 1:length])
        near(got[1], lse[length - 1:length], lse_bound[length - 1:length])


def test_scales_beyond_their_range_are_refused():
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device=DEV)
    pool, table, lens = torch.zeros(1, 16, 2, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(4, 1, dtype=torch.int32, device=DEV), torch.ones(
        4, dtype=torch.int32, device=DEV)
    for scale in (2.5e38, 3e38, 1e39, 1e-46):   # scale log2(e) infinite, the scale itself, the scale zero
        with pytest.raises(RuntimeError, match="positive"):
            mslk_amd.attention_prompt(q, q, q, offsets([4]).to(DEV), scale=scale)
        with pytest.raises(RuntimeError, match="positive"):
            mslk_amd.attention_decode(q, pool, pool, table, lens, scale=scale)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [64, 72, 80, 200])
def test_prompt_infinite_keys_and_values(d, causal):
    """Keys that score minus infinity weigh nothing; an infinite value of the last key makes its channel infinite where it is seen."""
    g = torch.Generator().manual_seed(d)
    n = 150
    q, k, v = (heads(g, n, 2, d, torch.bfloat16) for _ in range(3))
    q[:, :, -1] = q[:, :, -1].abs() + 1
    gone = torch.zeros(n, dtype=torch.bool)
    gone[10:20] = gone[70:140] = True
    visible = (causal_mask(n, n) if causal else torch.ones(n, n, dtype=torch.bool)) & ~gone
    out, lse, bound, lse_bound = attention(q, k, v, d ** -0.5, visible)
    k[gone, :, -1] = -math.inf
    v[n - 1, 0, 3] = math.inf
    out[visible[:, n - 1], 0, 3] = math.inf
    got = mslk_amd.attention_prompt(*(x.to(DEV) for x in (q, k, v)), offsets([n]).to(DEV), causal=causal, return_lse=True)
    near(got[0], out, bound)
    near(got[1], lse, lse_bound)


def test_prompt_strides_and_alignment():
    g = torch.Generator().manual_seed(7)
    t, hq, hkv, d = 210, 6, 2, 96
    fused = heads(g, t, hq + 2 * hkv, d, torch.bfloat16).to(DEV)
    q, k, v = fused[:, :hq], fused[:, hq:hq + hkv], fused[:, hq + hkv:]
    want = check_prompt(q.cpu(), k.cpu(), v.cpu(), [200, 10])
    cu = offsets([200, 10]).to(DEV)
    by_head = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    wide = [torch.zeros(*x.shape[:2], 2 * d, dtype=x.dtype, device=DEV)[..., :d].copy_(x) for x in (q, k, v)]
    odd = [torch.zeros(*x.shape[:2], d + 1, dtype=x.dtype, device=DEV)[..., 1:].copy_(x) for x in (q, k, v)]
    every_other = [torch.zeros(*x.shape[:2], 2 * d, dtype=x.dtype, device=DEV)[..., ::2].copy_(x) for x in (q, k, v)]
    for views in ((q, k, v), by_head, wide, odd, every_other):
        out, lse = mslk_amd.attention_prompt(*views, cu, return_lse=True)
        assert torch.equal(out.cpu(), want[0].cpu()) and torch.equal(lse.cpu(), want[1].cpu())
    one = mslk_amd.attention_prompt(q, k[:, :1].expand(-1, 6, -1), v[:, :1].expand(-1, 6, -1), cu)   # a head read six times
    assert torch.equal(one, mslk_amd.attention_prompt(q, k[:, :1], v[:, :1], cu))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [64, 72, 128, 200])
@pytest.mark.parametrize("t", [1, 40, 70])
def test_prompt_keys_and_values_that_share_memory(t, d, causal):
    """One key for more queries than a wave holds; a key and a value repeated for all tokens; rows that overlap.  An infinite value
    makes its channel infinite where it is seen, not NaN."""
    g = torch.Generator().manual_seed(t + d)
    n = 200
    q, row = heads(g, n, 4, d, torch.bfloat16), heads(g, 1, 2, d, torch.bfloat16)
    row[0, 1, 3] = math.inf
    flat = torch.randn(2, 8 * t + d, generator=g).bfloat16()
    flat[1, 8 * (t - 1) + 9] = math.inf
    sliding = [flat.to(DEV).as_strided((t, 2, d), (8, 8 * t + d, 1)), flat.as_strided((t, 2, d), (8, 8 * t + d, 1))]
    for on_gpu, rows in ((row.to(DEV).expand(t, -1, -1), row.expand(t, -1, -1)), sliding):
        seen = (causal_mask(n, t) if causal else torch.ones(n, t, dtype=torch.bool))
        # scores of finite keys; values: the finite ones, and infinite where such a value is seen
        key = torch.where(rows.isinf(), 0, rows)
        out, lse, bound, lse_bound = attention(q, key, key, d ** -0.5, seen)
        wild = torch.einsum("nt,thd->nhd", seen.float(), rows.isinf().float()).repeat_interleave(2, 1) > 0
        out[wild] = math.inf
        got = mslk_amd.attention_prompt(q.to(DEV), key.to(DEV) if rows is sliding[1] else torch.where(row.isinf(), 0, row).to(DEV).expand(t, -1, -1),
                                        on_gpu, offsets([n]).to(DEV), offsets([t]).to(DEV), causal=causal, return_lse=True)
        near(got[0], out, bound)
        near(got[1], lse, lse_bound)


def test_prompt_refuses_overlapping_rows_through_the_c_interface():
    import ctypes
    from mslk_amd import _lib
    x, out = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(4, 2, 64, dtype=torch.bfloat16, device=DEV)
    lse, cu = torch.zeros(4, 2, device=DEV), offsets([4]).to(DEV)
    rows = lambda stride: ctypes.byref(_lib.Heads(x.data_ptr(), stride, 64))   # noqa: E731
    def call(k_stride, v_stride):
        return _lib.lib().mslk_amd_attention_prompt(rows(128), rows(k_stride), rows(v_stride), 0, 4, 4, 2, 2, 64, cu.data_ptr(), None, 1, 1, 1.0,
                                                    out.data_ptr(), lse.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert call(0, 128) != 0 and call(128, 56) != 0
    assert call(128, 128) == 0 and call(64, 64) == 0
    torch.cuda.synchronize()


def test_prompt_long():
    """16 thousand keys: against the definition on the GPU in 64 bits, a few of the rows."""
    g = torch.Generator().manual_seed(8)
    n = 16391
    q, k, v = heads(g, n, 1, 128, torch.bfloat16), heads(g, n, 1, 128, torch.bfloat16), heads(g, n, 1, 128, torch.bfloat16)
    out, lse = mslk_amd.attention_prompt(*(x.to(DEV) for x in (q, k, v)), offsets([n]).to(DEV), return_lse=True)
    rows = torch.tensor([0, 1, 63, 64, 5000, 8191, 8192, 16255, 16256, 16383, 16390])
    want = attention(q[rows], k, v, 128 ** -0.5, torch.arange(n)[None] <= rows[:, None])
    near(out[rows.to(DEV)], want[0], want[2])
    near(lse[rows.to(DEV)], want[1], want[3])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [40, 64, 80, 96, 128, 160, 192, 256])
def test_prompt_many_heads(d, dtype):
    """As many heads as fill the machine: the larger blocks of queries."""
    g = torch.Generator().manual_seed(d)
    lens = [257, 1, 77]
    q, k, v = heads(g, sum(lens), 120, d, dtype), heads(g, sum(lens), 8, d, dtype), heads(g, sum(lens), 8, d, dtype)
    v[250, 0, 3] = math.nan if dtype == torch.float16 else math.inf      # hidden from all rows of its head but the last of a sequence
    k[257 + 1 + 60, 1, 5] = math.inf
    seen = [x.clone() for x in (k, v)]
    seen[0][257 + 1 + 60:, 1] = 0
    seen[1][250:257, 0] = 0
    out, lse = mslk_amd.attention_prompt(q.to(DEV), k.to(DEV), v.to(DEV), offsets(lens).to(DEV), return_lse=True)
    at = 0
    for n in lens:
        want = attention(q[at:at + n], seen[0][at:at + n], seen[1][at:at + n], d ** -0.5, causal_mask(n, n))
        upto = n - 7 if n == 257 else 60 if n == 77 else n               # rows in front of the wild ones
        for got, w, bound in ((out, want[0], want[2]), (lse, want[1], want[3])):
            near(got[at:at + upto], w[:upto], bound[:upto])
        at += n


@pytest.mark.parametrize("hq,hkv", [(2, 1), (8, 8), (48, 16)])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_ragged_batches(hq, hkv, causal):
    """2 to 65 sequences of any lengths, few and many heads: whichever order the blocks of queries are taken in, each comes once."""
    g = torch.Generator().manual_seed(hq)
    for n in (2, 9, 64, 65):
        lens = (torch.rand(n, generator=g) ** 4 * 400).int().tolist()
        lens_k = [max(x + int(e) - 90, 0) for x, e in zip(lens, torch.randint(0, 200, (n,), generator=g))]
        q = heads(g, sum(lens), hq, 64, torch.bfloat16)
        k, v = heads(g, sum(lens_k), hkv, 64, torch.bfloat16), heads(g, sum(lens_k), hkv, 64, torch.bfloat16)
        check_prompt(q, k, v, lens, lens_k, causal)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("step", [0.05, 0.11, 0.12, 0.5, -0.11])
def test_prompt_scores_that_creep_up(d, step):
    """Each key's score lies `step` powers of two above the last one's: a tile's maximum rises by less and by more than what the
    weights may grow by before they are taken from another reference."""
    g = torch.Generator().manual_seed(int(step * 100) + d)
    n = 333
    q, k, v = heads(g, n, 2, d, torch.bfloat16), heads(g, n, 1, d, torch.bfloat16) / 64, heads(g, n, 1, d, torch.bfloat16)
    q[:, :, 0] = 1
    k[:, :, 0] = (step * math.log(2) * torch.arange(n)[:, None]).bfloat16()
    check_prompt(q, k, v, [n], scale=1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq", [4, 104])
def test_scores_whose_rounding_is_many_powers_of_two(hq, d, dtype):
    """Scores of 10^6 to 10^37: one key in each half of the sequence scores twice what the others do, so the output is its value
    (up to the weight's one rounding) and lse its score, with the rounding of scale log2(e) and of two products."""
    g = torch.Generator().manual_seed(34)
    n = 300
    q, k, v = torch.zeros(n, hq, d, dtype=dtype), torch.zeros(n, 4, d, dtype=dtype), heads(g, n, 4, d, dtype)
    q[:, :, 0] = 1031
    for scale in [float(x) for x in 10 ** (1 + 4 * torch.rand(6, generator=g))] + ([1e13, 1e30] if dtype == torch.bfloat16 else []):
        for sign in (1, -1):
            k[:, :, 0] = sign * (1000 + 8 * torch.rand(n, 1, generator=g)) * (1 if sign > 0 else 3)
            k[40, :, 0] = sign * 2003
            k[211, :, 0] = sign * (4007 if sign > 0 else 1001)
            winner = torch.where(torch.arange(n) >= 211, 211, 40)
            out, lse = mslk_amd.attention_prompt(*(x.to(DEV) for x in (q, k, v)), offsets([n]).to(DEV), scale=scale, return_lse=True)
            score = (q.double()[:, :, :1] * k.double()[winner][:, :, :1].repeat_interleave(hq // 4, 1))[..., 0] * scale
            value = v.double()[winner].repeat_interleave(hq // 4, 1)
            seen = slice(40, n)
            near(out[seen], value[seen], (2 * ROUND[dtype] * value.abs())[seen], f"{scale}")
            near(lse[seen], score[seen], 2.0 ** -21 * score[seen].abs(), f"lse, {scale}")
            cache = Cache(g, [n], 4, d, 16, dtype, rows=[[k], [v]])
            got = mslk_amd.attention_decode(q[:1].to(DEV), *cache.on_gpu(), scale=scale, return_lse=True)
            near(got[0], value[n - 1:], 2 * ROUND[dtype] * value[n - 1:].abs())
            near(got[1], score[n - 1:], 2.0 ** -21 * score[n - 1:].abs())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("tokens,hq", [(16, 4), (300, 104)])
def test_prompt_equal_scores_weigh_the_same_in_every_tile(tokens, hq, d, dtype):
    """Scores that are all the same, however large: the reference stays, so the sums of the first tile may not fade until the last.
    Values of 1 in the first half of the keys and -1 in the second add up to zero, exactly: a weight of 11 bits times up to 2^13 keys
    fits 24.  lse: the rounding of scale log2(e) and of two products, 2^-21 of it, and 256 sums of a row in 32 bits, 2^-14."""
    n = 16384
    scores = torch.tensor([50.0, 700.0, -300.0, 37.0])
    q, k, v = torch.zeros(tokens, hq, d, dtype=dtype), torch.zeros(n, 4, d, dtype=dtype), torch.ones(n, 4, d, dtype=dtype)
    q[:, :, 0] = 1
    k[:, :, 0] = scores.to(dtype)
    v[n // 2:] = -1
    cu, cu_k = offsets([tokens]).to(DEV), offsets([n]).to(DEV)
    for scale in (1.0, 0.7):
        out, lse = mslk_amd.attention_prompt(*(x.to(DEV) for x in (q, k, v)), cu, cu_k, causal=False, scale=scale, return_lse=True)
        assert out.float().abs().max() <= 2.0 ** -20
        want = (scores.double() * torch.tensor(scale).double() + math.log(n)).repeat_interleave(hq // 4).expand(tokens, -1)
        near(lse, want, 2.0 ** -21 * want.abs() + 2.0 ** -14)


def test_prompt_many_sequences_and_repeat():
    g = torch.Generator().manual_seed(9)
    lens = torch.randint(0, 9, (300,), generator=g).tolist()
    q, k, v = heads(g, sum(lens), 2, 64, torch.bfloat16), heads(g, sum(lens), 2, 64, torch.bfloat16), heads(g, sum(lens), 2, 64, torch.bfloat16)
    first = check_prompt(q, k, v, lens)
    again = check_prompt(q, k, v, lens)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


# ---------------------------------------------------------------------------------------------------------------------
# paged caches
# ---------------------------------------------------------------------------------------------------------------------
class Cache:
    """A pool of pages in random order, filled with keys and values [len, hkv, d] of each sequence; everything no key needs is NaN."""

    def __init__(self, g, lens, hkv, d, page, dtype, fp8=False, extra=2, rows=None):
        self.lens, self.page, self.fp8 = lens, page, fp8
        counts = [-(-n // page) for n in lens]
        pages = sum(counts) + 3
        self.table = torch.full((len(lens), max(counts + [0]) + extra), -1, dtype=torch.int32)
        free = torch.randperm(pages, generator=g).tolist()
        for b, c in enumerate(counts):
            for i in range(c):
                self.table[b, i] = free.pop()
        self.k = [heads(g, n, hkv, d, dtype) for n in lens] if rows is None else rows[0]
        self.v = [heads(g, n, hkv, d, dtype) for n in lens] if rows is None else rows[1]
        self.pools, self.scales = [], [None, None]
        for which, rows_of in enumerate((self.k, self.v)):
            pool = torch.full((pages, page, hkv, d), math.nan).to(F8 if fp8 else dtype)
            scale = torch.full((pages, page, hkv), math.nan)
            for b, rows_b in enumerate(rows_of):
                if fp8:
                    amax = rows_b.float().abs().amax(-1).clamp(min=1e-12)
                    codes, sc = (rows_b.float() * (448.0 / amax)[..., None]).to(F8), amax / 448.0
                    rows_of[b] = codes.double() * sc.double()[..., None]
                for t in range(len(rows_b)):
                    at = (int(self.table[b, t // page]), t % page)
                    if fp8:
                        pool.view(torch.uint8)[at], scale[at] = codes[t].view(torch.uint8), sc[t]
                    else:
                        pool[at] = rows_b[t]
            self.pools.append(pool)
            if fp8:
                self.scales[which] = scale

    def on_gpu(self):
        scales = [None if s is None else s.to(DEV) for s in self.scales]
        return [p.to(DEV) for p in self.pools] + [self.table.to(DEV), torch.tensor(self.lens, dtype=torch.int32).to(DEV)] + scales


def check_decode(q, cache, scale=None, got=None):
    if got is None:
        got = mslk_amd.attention_decode(q.to(DEV), *cache.on_gpu(), scale=scale, return_lse=True)
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    for b, n in enumerate(cache.lens):
        out, lse, bound, lse_bound = attention(q[b:b + 1], cache.k[b], cache.v[b], scale, torch.ones(1, n, dtype=torch.bool))
        near(got[0][b:b + 1], out, bound, f"sequence {b} of {n}")
        near(got[1][b:b + 1], lse, lse_bound, f"lse of sequence {b} of {n}")
    return got


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [8, 64, 72, 80, 96, 128, 136, 192, 256])
def test_decode_head_dimensions(d, dtype, fp8):
    g = torch.Generator().manual_seed(d)
    lens = [1, 40, 300]
    check_decode(heads(g, 3, 8, d, dtype), Cache(g, lens, 2, d, 16, dtype, fp8))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("lens", [[0], [1], [0, 0, 3], [31, 32, 33], [127, 128, 129], [255, 0, 257, 1], [1] * 130, [1000, 1, 2000], [4097]])
def test_decode_lengths(lens, fp8):
    g = torch.Generator().manual_seed(sum(lens))
    check_decode(heads(g, len(lens), 4, 64, torch.bfloat16), Cache(g, lens, 2, 64, 16, torch.bfloat16, fp8))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("d", [64, 128, 200])
@pytest.mark.parametrize("lens", [[0], [1], [0, 0, 3], [31, 32, 33], [127, 128, 129], [255, 0, 257, 1], [1] * 130, [1000, 1, 700], [65] * 70 + [0] * 70])
def test_decode_lengths_in_wide_tables(lens, d, fp8):
    """Tables with room for many more keys: how the work is divided goes by what they could hold."""
    g = torch.Generator().manual_seed(sum(lens) + d)
    check_decode(heads(g, len(lens), 6, d, torch.bfloat16), Cache(g, lens, 2, d, 16, torch.bfloat16, fp8, extra=100))


@pytest.mark.parametrize("sequences,hkv,longest", [(3, 1, 120), (3, 1, 200), (40, 4, 200), (200, 1, 500), (300, 2, 1000), (140, 8, 1030)])
def test_decode_batches_of_short_caches(sequences, hkv, longest):
    g = torch.Generator().manual_seed(longest)
    lens = torch.randint(0, longest, (sequences,), generator=g).tolist()
    lens[0] = longest
    check_decode(heads(g, sequences, 2 * hkv, 64, torch.float16), Cache(g, lens, hkv, 64, 8, torch.float16, extra=0))


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (15, 1), (16, 1), (17, 1), (40, 1), (5, 5), (64, 8), (34, 2), (48, 16)])
def test_decode_head_layouts(hq, hkv):
    g = torch.Generator().manual_seed(hq)
    lens = [200, 33, 0]
    check_decode(heads(g, 3, hq, 64, torch.bfloat16), Cache(g, lens, hkv, 64, 32, torch.bfloat16))


@pytest.mark.parametrize("page", [1, 2, 3, 5, 7, 16, 33, 64, 100, 128, 1000])
def test_decode_page_sizes(page):
    g = torch.Generator().manual_seed(page)
    lens = [137, 64, 999, 5]
    check_decode(heads(g, 4, 4, 64, torch.float16), Cache(g, lens, 2, 64, page, torch.float16))
    check_decode(heads(g, 4, 4, 64, torch.float16), Cache(g, lens, 2, 64, page, torch.float16, fp8=True))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("extra", [2, 5000])
@pytest.mark.parametrize("lens", [[0], [0, 40, 0, 33, 0], [0] * 3, [7, 0]])
def test_decode_empty_sequences_with_pages_of_one_key(lens, extra, fp8):
    """A sequence without keys reads nothing of its table, whose entry of a key -1 would lie in front of it: the first table row,
    rows in between and one for all sequences, few keys of room (a head block per wave) and much of it (equal parts)."""
    g = torch.Generator().manual_seed(sum(lens))
    cache = Cache(g, lens, 2, 64, 1, torch.bfloat16, fp8, extra=extra)
    q = heads(g, len(lens), 4, 64, torch.bfloat16)
    check_decode(q, cache)
    if not any(lens):
        k, v, table, kv_lens, ks, vs = cache.on_gpu()
        for t in (table[:1].expand(len(lens), -1), torch.zeros(len(lens), 0, dtype=torch.int32, device=DEV)):
            out, lse = mslk_amd.attention_decode(q.to(DEV), k, v, t, kv_lens, ks, vs, return_lse=True)
            assert (out == 0).all() and (lse == -math.inf).all()


def test_decode_scores_far_apart_and_scales_far_apart():
    g = torch.Generator().manual_seed(11)
    lens = [700, 90]
    rows = [[heads(g, n, 2, 64, torch.float16) for n in lens] for _ in range(2)]
    rows[0][0][100:110] *= 60
    rows[0][0][500:] *= 0.01
    rows[1][0][::3] *= 2.0 ** -8
    rows[1][0][::7] = 0
    rows[1][1] *= 2.0 ** -12
    q = heads(g, 2, 6, 64, torch.float16)
    for fp8 in (False, True):
        for scale in (None, 4.0):
            check_decode(q, Cache(g, lens, 2, 64, 16, torch.float16, fp8, rows=[[x.clone() for x in r] for r in rows]), scale)


def test_decode_strides():
    """Pools by head, q out of a projection's output, a table wider than it needs to be with a row stride."""
    g = torch.Generator().manual_seed(12)
    cache = Cache(g, [300, 17], 2, 128, 16, torch.bfloat16)
    fused = heads(g, 2, 12, 128, torch.bfloat16).to(DEV)
    q = fused[:, :8]
    k, v, table, lens, _, _ = cache.on_gpu()
    want = check_decode(q.cpu(), cache)
    by_head = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v)]
    mixed = [k.transpose(0, 1).contiguous().transpose(0, 1), v]
    wide = torch.full((2, table.shape[1] + 50), -7, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    for pools, t in ((by_head, table), (mixed, table), ((k, v), wide), ((k, v), wide[:, :table.shape[1]])):
        out, lse = mslk_amd.attention_decode(q, *pools, t, lens, return_lse=True)
        check_decode(q.cpu(), cache, got=(out, lse))
        if t.shape == table.shape:
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    shifted = torch.zeros(2, 8, 129, dtype=torch.bfloat16, device=DEV)[..., 1:].copy_(q)
    assert torch.equal(mslk_amd.attention_decode(shifted, k, v, table, lens), want[0])
    fp8 = Cache(torch.Generator().manual_seed(13), [300, 17], 2, 128, 16, torch.bfloat16, True)
    k, v, table, lens, ks, vs = fp8.on_gpu()
    want = check_decode(q.cpu(), fp8)
    out = mslk_amd.attention_decode(q, *(x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v)), table, lens,
                                    ks.permute(2, 0, 1).contiguous().permute(1, 2, 0), vs)
    assert torch.equal(out, want[0])


def test_decode_keys_without_a_page_give_nan():
    g = torch.Generator().manual_seed(14)
    cache = Cache(g, [100, 50, 30, 20], 2, 64, 16, torch.bfloat16)
    q = heads(g, 4, 4, 64, torch.bfloat16)
    k, v, table, lens, _, _ = cache.on_gpu()
    table[0, 3] = -1                    # inside the sequence
    table[1, 0] = k.shape[0]            # no such page
    lens[2] = table.shape[1] * 16 + 9   # beyond the table
    lens[3] = -5                        # none
    out, lse = mslk_amd.attention_decode(q.to(DEV), k, v, table, lens, return_lse=True)
    assert torch.isnan(out[:3]).all() and torch.isnan(lse[:3]).all()
    assert (out[3] == 0).all() and (lse[3] == -math.inf).all()


def test_decode_wild_values_touch_their_sequence_only():
    g = torch.Generator().manual_seed(15)
    rows = [[heads(g, n, 2, 64, torch.bfloat16) for n in (100, 70)] for _ in range(2)]
    q = heads(g, 2, 4, 64, torch.bfloat16)
    rows[1][0][33, 1, 2] = math.inf
    rows[1][0][34, 0, 3] = math.nan
    out = mslk_amd.attention_decode(q.to(DEV), *Cache(g, [100, 70], 2, 64, 16, torch.bfloat16, rows=rows).on_gpu()).cpu()
    assert (out[0, 2:, 2] == math.inf).all() and torch.isnan(out[0, :2, 3]).all()
    assert torch.isfinite(out).sum() == out.numel() - 4


@pytest.mark.parametrize("d", [64, 72, 80, 136, 200])
def test_decode_infinite_keys_and_values(d):
    """Keys that score minus infinity weigh nothing; an infinite value of the last key makes its channel infinite, not NaN."""
    g = torch.Generator().manual_seed(d)
    lens = [33, 100, 2500]
    rows = [[heads(g, n, 2, d, torch.bfloat16) for n in lens] for _ in range(2)]
    q = heads(g, 3, 4, d, torch.bfloat16)
    q[:, :, -1] = q[:, :, -1].abs() + 1
    want = []
    for b, n in enumerate(lens):
        gone = (torch.arange(n) >= n // 3) & (torch.arange(n) < n // 3 + 20)
        want.append(attention(q[b:b + 1], rows[0][b], rows[1][b], d ** -0.5, ~gone[None]))
        rows[0][b][gone, :, -1] = -math.inf
        rows[1][b][n - 1, 1, 5] = math.inf
        want[b][0][0, 2:, 5] = math.inf
    got = mslk_amd.attention_decode(q.to(DEV), *Cache(g, lens, 2, d, 16, torch.bfloat16, rows=rows).on_gpu(), return_lse=True)
    for b, (out, lse, bound, lse_bound) in enumerate(want):
        near(got[0][b:b + 1], out, bound)
        near(got[1][b:b + 1], lse, lse_bound)


def test_decode_with_room_for_2_to_the_30_keys():
    """The most that a page table may have room for; a length beyond it gives NaN as any that the table cannot hold."""
    g = torch.Generator().manual_seed(17)
    cache = Cache(g, [700, 90], 1, 64, 1024, torch.bfloat16)
    q = heads(g, 2, 2, 64, torch.bfloat16)
    k, v, table, lens, _, _ = cache.on_gpu()
    wide = torch.full((2, 1 << 20), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    check_decode(q, cache, got=mslk_amd.attention_decode(q.to(DEV), k, v, wide, lens, return_lse=True))
    with pytest.raises(RuntimeError, match="2.30 keys"):
        mslk_amd.attention_decode(q.to(DEV), k, v, torch.zeros(1, (1 << 20) + 1, dtype=torch.int32, device=DEV).expand(2, -1), lens)


@pytest.mark.parametrize("hkv,room", [(1032, 4), (264, 1040)])
def test_decode_with_more_workgroups_than_one_line_of_a_grid(hkv, room):
    """65535 sequences of many heads: more than 2^32 work-items, a head block per wave (little room) and in the join (much of it),
    against the same call on parts of the sequences.  Values of one sign and about one size, so that the bound of a call is (2 u + 2^-16) |out|
    (scores of 8 channels: their errors lie below 2^-18), and of two calls twice that."""
    g = torch.Generator(DEV).manual_seed(18)
    b, d, page = 65535, 8, 4
    k, v = torch.randn(300, page, hkv, d, generator=g, device=DEV).bfloat16(), (torch.rand(300, page, hkv, d, generator=g, device=DEV) + 0.5).bfloat16()
    q = torch.randn(b, hkv, d, generator=g, device=DEV, dtype=torch.bfloat16)
    table = torch.randint(0, 300, (b, room // page), generator=g, device=DEV, dtype=torch.int32)
    lens = torch.randint(0, 4, (b,), generator=g, device=DEV, dtype=torch.int32)
    lens[::256] = room
    out, lse = mslk_amd.attention_decode(q, k, v, table, lens, return_lse=True)
    for at in range(0, b, 8192):
        part = slice(at, min(at + 8192, b))
        want, want_lse = mslk_amd.attention_decode(q[part], k, v, table[part], lens[part], return_lse=True)
        empty = lens[part] == 0
        assert (out[part][empty] == 0).all() and (lse[part][empty] == -math.inf).all()
        got, want = out[part][~empty].float(), want[~empty].float()
        assert ((got - want).abs() <= 2 * (2.0 ** -7 + 2.0 ** -16) * want).all()
        assert ((lse[part] - want_lse)[~empty].abs() <= 2.0 ** -17 * (1 + want_lse[~empty].abs())).all()
    del q, out, lse
    torch.cuda.empty_cache()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,lens,extra", [(64, [300, 40], 2), (128, [5000, 1], 2), (80, [90, 33], 0), (256, [700, 64], 100)])
def test_decode_weights_are_not_rounded_to_16_bits(d, lens, extra, dtype, fp8):
    """The output is off by its own rounding and by its share of the weights' error: 2^-15 where they are two numbers of 8 bits, 2^-20 where
    they are two of 11, and the scores' error in fp32.  (One number each, 2^-8 and 2^-11, shows where values cancel out.)"""
    g = torch.Generator().manual_seed(d)
    cache = Cache(g, lens, 2, d, 16, dtype, fp8, extra=extra)
    q = heads(g, 2, 8, d, dtype)
    got = mslk_amd.attention_decode(q.to(DEV), *cache.on_gpu(), return_lse=True)
    for b, n in enumerate(lens):
        everything = torch.ones(1, n, dtype=torch.bool)
        out, _, _, two_delta = attention(q[b:b + 1], cache.k[b], cache.v[b], d ** -0.5, everything)
        size = attention(q[b:b + 1], cache.k[b], cache.v[b].abs(), d ** -0.5, everything)[0]   # sum of weight times |value|
        weights = 2.0 ** -15 if dtype == torch.bfloat16 else 2.0 ** -20
        near(got[0][b:b + 1], out, ROUND[dtype] * out.abs() + (weights + two_delta[..., None]) * size + 2.0 ** -25, f"sequence {b} of {n}")


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_decode_infinite_values_of_small_weights(dtype, fp8):
    """A value of infinity makes its channel infinite for every weight down to 2^-20 of the largest, not NaN, and the others stay."""
    g = torch.Generator().manual_seed(36)
    n, d = 120, 64
    k, v = torch.zeros(n, 1, d, dtype=dtype), heads(g, n, 1, d, dtype)
    k[:, 0, 0] = -(torch.arange(n) / 6.0).to(dtype)          # weights of 2^(-i / 6)
    q = torch.zeros(n, 1, d, dtype=dtype)
    q[:, 0, 0] = 1
    cache = Cache(g, [n], 1, d, 16, dtype, fp8, extra=0, rows=[[k], [v]])   # (few keys of room: not cut, one reference)
    kc, vc, table, lens, ks, vs = cache.on_gpu()
    want = mslk_amd.attention_decode(q[:1].to(DEV), kc, vc, table, lens, ks, vs, scale=math.log(2.0))
    for i in range(n):
        pools = vc.clone()
        at = (int(cache.table[0, i // 16]), i % 16, 0, 7)
        scales = vs
        if fp8:                                              # e4m3 has no infinity: a row of an infinite scale, its codes not zero
            pools.view(torch.uint8)[at[:3]] = 0x38
            scales = vs.clone()
            scales[at[:3]] = math.inf
        else:
            pools[at] = math.inf
        out = mslk_amd.attention_decode(q[:1].to(DEV), kc, pools, table, lens, ks, scales, scale=math.log(2.0))
        if fp8:
            assert (out == math.inf).all(), i
        else:
            assert out[0, 0, 7] == math.inf, i
            assert torch.equal(out[..., torch.arange(d) != 7], want[..., torch.arange(d) != 7]), i


def test_decode_long_and_offsets_beyond_32_bits():
    """A pool of more than 2^32 bytes whose used pages lie at both ends."""
    g = torch.Generator().manual_seed(16)
    pages, page, hkv, d = 36000, 64, 8, 128      # 4.7 GB of keys
    pool = [torch.zeros(pages, page, hkv, d, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    n = 5000
    rows = [heads(g, n, hkv, d, torch.bfloat16) for _ in range(2)]
    ids = torch.cat([torch.arange(pages - 40, pages), torch.arange(39)])[torch.randperm(79, generator=g)].to(torch.int32)
    for p, r in zip(pool, rows):
        flat = torch.zeros(79 * page, hkv, d, dtype=torch.bfloat16)
        flat[:n] = r
        p[ids.long().to(DEV)] = flat.view(79, page, hkv, d).to(DEV)
    q = heads(g, 1, 16, d, torch.bfloat16)
    out, lse = mslk_amd.attention_decode(q.to(DEV), *pool, ids[None].to(DEV), torch.tensor([n], dtype=torch.int32, device=DEV), return_lse=True)
    want = attention(q, *rows, d ** -0.5, torch.ones(1, n, dtype=torch.bool))
    near(out, want[0], want[2])
    near(lse, want[1], want[3])


# ---------------------------------------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------------------------------------
def rotary_table(positions, r):
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def rotated(x, table, positions, interleaved):
    """(rotated rows, bound of their fp32 arithmetic) in 64 bits."""
    x = x.double()
    half = table.shape[1] // 2
    cos, sin = table.double()[positions].chunk(2, -1)
    cos, sin = cos[:, None], sin[:, None]
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = x[..., first], x[..., second]
    out, slack = x.clone(), torch.zeros_like(x)
    out[..., first], out[..., second] = a * cos - b * sin, b * cos + a * sin
    slack[..., first] = slack[..., second] = 2.0 ** -22 * (a.abs() + b.abs())
    return out, slack


def check_append(g, new, total, hq, hkv, d, page, dtype, fp8=False, r=None, interleaved=False, packed=True):
    """`new` tokens at the end of sequences of `total` keys; everything else of the cache has to stay as it is."""
    t = sum(new)
    fused = heads(g, t, hq + 2 * hkv, d, dtype)
    q, k, v = fused[:, :hq], fused[:, hq:hq + hkv], fused[:, hq + hkv:]
    r = d if r is None else r
    table = rotary_table(max(total), r) if r else None
    cache = Cache(g, total, hkv, d, page, dtype, fp8)
    pools, scales = [p.to(DEV) for p in cache.pools], [None if s is None else s.to(DEV) for s in cache.scales]
    whole = fused.to(DEV)
    out = mslk_amd.append_kv(whole[:, :hq], whole[:, hq:hq + hkv], whole[:, hq + hkv:], *pools, cache.table.to(DEV),
                             torch.tensor(total, dtype=torch.int32).to(DEV), offsets(new).to(DEV) if packed else None,
                             None if table is None else table.to(DEV), interleaved, *scales)
    positions = torch.tensor([n - m + i for m, n in zip(new, total) for i in range(m)], dtype=torch.long)
    seqs = torch.tensor([b for b, m in enumerate(new) for _ in range(m)], dtype=torch.long)
    u = ROUND[dtype]
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0   # half a subnormal's spacing

    def turn(x):
        return rotated(x, table, positions, interleaved) if r else (x.double(), torch.zeros(x.shape, dtype=torch.float64))

    want, slack = turn(q)
    near(out, want, u * want.abs() + slack + tiny, "q")
    at = (cache.table[seqs, positions // page].long(), positions % page)
    for name, x, pool, scale, before, scale_before in (("k", k, pools[0], scales[0], cache.pools[0], cache.scales[0]),
                                                        ("v", v, pools[1], scales[1], cache.pools[1], cache.scales[1])):
        want, slack = turn(x) if name == "k" else (x.double(), torch.zeros(x.shape, dtype=torch.float64))
        pool = pool.cpu()
        if fp8:
            scale = scale.cpu()
            amax = want.abs().amax(-1).clamp(min=1e-12)
            near(scale[at], amax / 448, 2.0 ** -22 * amax / 448 + slack.amax(-1) / 448, name + " scale")
            codes = want * (448 / amax)[..., None]
            # e4m3: half a step, 2^-4 relative or 2^-10 below 2^-6; a code that lies near a tie may go either way
            near(pool[at].float(), codes, codes.abs() * (2.0 ** -4 + 2.0 ** -20) + 2.0 ** -10 + slack * (449 / amax)[..., None], name)
            scale_before = scale_before.clone()
            scale_before[at] = scale[at]
            assert torch.equal(scale.view(torch.int32), scale_before.view(torch.int32)), name + ": a scale elsewhere changed"
            kind = torch.uint8
        else:
            near(pool[at], want, u * want.abs() + slack + tiny, name)
            if name == "v":
                assert torch.equal(pool[at], x)
            kind = torch.int16
        before = before.clone()
        before.view(kind)[at] = pool.view(kind)[at]
        assert torch.equal(pool.view(kind), before.view(kind)), name + ": a row elsewhere changed"


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,r", [(8, 8), (64, 64), (80, 80), (80, 40), (96, 48), (128, 128), (128, 64), (128, 4), (128, 10), (128, 0), (192, 192),
                                 (256, 256), (256, 2), (256, 254), (72, 72)])
def test_append_head_dimensions(d, r, dtype, fp8):
    for interleaved in (False, True):
        check_append(torch.Generator().manual_seed(d + r), [3, 0, 9], [10, 4, 9], 4, 2, d, 16, dtype, fp8, r, interleaved)


@pytest.mark.parametrize("new,total,packed", [([1], [1], False), ([1] * 5, [1, 17, 16, 300, 33], False), ([1, 0, 1], [4, 2, 65], True),
                                              ([40, 1, 200], [40, 500, 333], True), ([0, 0], [3, 5], True)])
@pytest.mark.parametrize("page", [1, 7, 16, 128])
def test_append_lengths(new, total, packed, page):
    check_append(torch.Generator().manual_seed(page), new, total, 6, 3, 64, page, torch.bfloat16, packed=packed)


def test_append_many_sequences():
    g = torch.Generator().manual_seed(20)
    new = torch.randint(0, 4, (333,), generator=g).tolist()
    check_append(g, new, [n + 5 * (i % 7) for i, n in enumerate(new)], 2, 1, 64, 16, torch.float16, True)


def test_append_padding_and_tokens_without_a_place():
    g = torch.Generator().manual_seed(21)
    cache = Cache(g, [20, 20, 20, 20], 2, 64, 16, torch.bfloat16)
    q, k, v = (heads(g, 8, n, 64, torch.bfloat16).to(DEV) for n in (4, 2, 2))
    pools = [p.to(DEV) for p in cache.pools]
    before = [p.clone() for p in pools]
    table = cache.table.clone()
    table[1, 1] = 10 ** 6                                        # sequence 1: position 19 lies in a page that is not there
    lens = torch.tensor([1, 20, 1000, 41], dtype=torch.int32)    # 0: two tokens for one position; 2: beyond the table; 3: beyond rotary
    cu = torch.tensor([1, 3, 4, 5, 6], dtype=torch.int32)        # token 0, 6 and 7 belong to nobody
    out = mslk_amd.append_kv(q, k, v, *pools, table.to(DEV), lens.to(DEV), cu.to(DEV), rotary_table(40, 64).to(DEV)).cpu()
    assert (out[[0, 1, 6, 7]] == 0).all() and torch.isnan(out[3:6]).all()
    assert torch.equal(out[2], q[2].cpu())                       # position 0
    at = int(table[0, 0])
    for pool, was, rows in zip(pools, before, (k, v)):
        assert torch.equal(pool[at, 0], rows[2])
        was[at, 0] = rows[2]
        assert torch.equal(pool.view(torch.int16), was.view(torch.int16))


def test_append_zero_and_wild_rows_in_fp8():
    g = torch.Generator().manual_seed(22)
    cache = Cache(g, [3], 1, 64, 16, torch.bfloat16, True)
    k, v = heads(g, 3, 1, 64, torch.bfloat16), heads(g, 3, 1, 64, torch.bfloat16)
    v[0], v[1, 0, 7], v[2, 0, 9] = 0, math.nan, math.inf
    pools, scales = [p.to(DEV) for p in cache.pools], [s.to(DEV) for s in cache.scales]
    mslk_amd.append_kv(k.to(DEV), k.to(DEV), v.to(DEV), *pools, cache.table.to(DEV), torch.tensor([3], dtype=torch.int32, device=DEV),
                       offsets([3]).to(DEV), k_scale=scales[0], v_scale=scales[1])
    at = int(cache.table[0, 0])
    rows = pools[1][at, :3, 0].float().cpu() * scales[1][at, :3, 0].cpu()[:, None]
    assert (rows[0] == 0).all() and torch.isnan(rows[1, 7]) and torch.isnan(rows[2, 9])
    assert torch.isfinite(scales[0][at, :3]).all()


# ---------------------------------------------------------------------------------------------------------------------
# together; streams, graphs, refusals
# ---------------------------------------------------------------------------------------------------------------------
def test_a_prompt_and_its_decoding_agree():
    """Every token of a sequence decoded over the cache gives what the prompt gives."""
    g = torch.Generator().manual_seed(30)
    n, hq, hkv, d, page = 90, 4, 2, 64, 16
    q, k, v = heads(g, n, hq, d, torch.bfloat16).to(DEV), heads(g, n, hkv, d, torch.bfloat16).to(DEV), heads(g, n, hkv, d, torch.bfloat16).to(DEV)
    pools = [torch.zeros(6, page, hkv, d, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    table = torch.tensor([[5, 0, 3, 1, 4, 2]], dtype=torch.int32, device=DEV)
    cu = offsets([n]).to(DEV)
    turned = mslk_amd.append_kv(q, k, v, *pools, table, torch.tensor([n], dtype=torch.int32, device=DEV), cu, rotary_table(n, d).to(DEV))
    keys, values = (p[table[0].long()].flatten(0, 1)[:n].cpu() for p in pools)
    check_prompt(turned.cpu(), keys, values, [n], got=mslk_amd.attention_prompt(turned, keys.to(DEV), values.to(DEV), cu, return_lse=True))
    lens = torch.arange(1, n + 1, dtype=torch.int32, device=DEV)
    got = mslk_amd.attention_decode(turned, *pools, table.expand(n, -1), lens, return_lse=True)
    check_prompt(turned.cpu(), keys, values, [n], got=got)


def test_other_stream():
    g = torch.Generator().manual_seed(31)
    cache = Cache(g, [500, 3], 2, 128, 16, torch.bfloat16)
    q = heads(g, 2, 8, 128, torch.bfloat16)
    on_gpu, q_gpu = cache.on_gpu(), q.to(DEV)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = mslk_amd.attention_decode(q_gpu, *on_gpu, return_lse=True)
        p = mslk_amd.attention_prompt(q_gpu, q_gpu, q_gpu, offsets([2]).to(DEV), return_lse=True)
    stream.synchronize()
    check_decode(q, cache, got=got)
    check_prompt(q, q, q, [2], got=p)


def test_graph_follows_lengths_and_tables():
    """One captured decode step replayed with other lengths, pages and tokens in the same buffers, against eager calls."""
    g = torch.Generator().manual_seed(32)
    hq, hkv, d, page, b = 8, 2, 128, 16, 3
    pools = [torch.randn(64, page, hkv, d, generator=g).bfloat16().to(DEV) for _ in range(2)]
    fused = torch.zeros(b, hq + 2 * hkv, d, dtype=torch.bfloat16, device=DEV)
    table, lens = torch.zeros(b, 20, dtype=torch.int32, device=DEV), torch.ones(b, dtype=torch.int32, device=DEV)
    rotary = rotary_table(400, d).to(DEV)

    def step(pk, pv):
        q = mslk_amd.append_kv(fused[:, :hq], fused[:, hq:hq + hkv], fused[:, hq + hkv:], pk, pv, table, lens, rotary=rotary)
        return mslk_amd.attention_decode(q, pk, pv, table, lens, return_lse=True)

    step(*pools)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step(*pools)
    for i, new in enumerate(([1, 300, 17], [320, 0, 2], [128, 129, 5], [320, 320, 320])):
        fused.copy_(torch.randn(fused.shape, generator=g).bfloat16())
        table.copy_(torch.randperm(64, generator=g)[:60].view(b, 20).to(torch.int32))
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        copies = [p.clone() for p in pools]
        want = step(*copies)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1]), i
        assert all(torch.equal(x, y) for x, y in zip(pools, copies)), i


def test_prompt_in_a_graph():
    g = torch.Generator().manual_seed(33)
    q, k, v = (heads(g, 300, 4, 64, torch.bfloat16).to(DEV) for _ in range(3))
    cu = offsets([100, 200]).to(DEV)
    mslk_amd.attention_prompt(q, k, v, cu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = mslk_amd.attention_prompt(q, k, v, cu, return_lse=True)
    for lens in ([300, 0], [1, 299], [128, 100], [150, 150]):
        cu.copy_(offsets(lens))
        want = mslk_amd.attention_prompt(q, k, v, cu, return_lse=True)
        torch.cuda.synchronize()
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1]), lens


def test_empty_calls():
    q, k = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(0, 2, 64, dtype=torch.bfloat16, device=DEV)
    none = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert mslk_amd.attention_prompt(q, k, k, none).shape == (0, 4, 64)
    pool = torch.zeros(1, 16, 2, 64, dtype=torch.bfloat16, device=DEV)
    table, lens = torch.zeros(0, 3, dtype=torch.int32, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV)
    assert mslk_amd.attention_decode(q, pool, pool, table, lens).shape == (0, 4, 64)
    assert mslk_amd.append_kv(q, k, k, pool, pool, table, lens).shape == (0, 4, 64)
    some = torch.randn(5, 4, 64, device=DEV).bfloat16()   # no sequence at all
    out, lse = mslk_amd.attention_prompt(some, some[:, :2], some[:, :2], none, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    lens = torch.zeros(5, dtype=torch.int32, device=DEV)   # no page at all
    assert (mslk_amd.attention_decode(some, pool, pool, torch.zeros(5, 0, dtype=torch.int32, device=DEV), lens) == 0).all()


def test_refusals():
    q, k = torch.zeros(4, 4, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(4, 2, 64, dtype=torch.bfloat16, device=DEV)
    cu = offsets([4]).to(DEV)

    def refused(what, call, *args, **kwargs):
        with pytest.raises(RuntimeError, match=what):
            call(*args, **kwargs)

    prompt = mslk_amd.attention_prompt
    refused("GPU", prompt, q.cpu(), k.cpu(), k.cpu(), cu.cpu())
    refused("bfloat16 or float16", prompt, q.float(), k.float(), k.float(), cu)
    refused("same dtype", prompt, q, k.half(), k, cu)
    refused("shape", prompt, q[0], k, k, cu)
    refused("same shape", prompt, q, k, k[:3], cu)
    refused("same number of channels", prompt, q, k[..., :56], k[..., :56], cu)
    refused("multiple of the KV heads", prompt, q[:, :3], k, k, cu)
    refused("multiple of 8", prompt, q[..., :60], k[..., :60], k[..., :60], cu)
    refused("multiple of 8", prompt, *(torch.zeros(4, 2, 264, dtype=torch.bfloat16, device=DEV) for _ in range(3)), cu)
    refused("int32", prompt, q, k, k, cu.long())
    refused("as many keys", prompt, q, k[:3], k[:3], cu)
    refused("as many offsets", prompt, q, k, k, cu, offsets([2, 2]).to(DEV))
    for scale in (0.0, -1.0, math.nan, math.inf):
        refused("positive", prompt, q, k, k, cu, scale=scale)

    pool = torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16, device=DEV)
    codes, row_scale = torch.zeros(3, 16, 2, 64, device=DEV).to(F8), torch.ones(3, 16, 2, device=DEV)
    table, lens = torch.zeros(4, 2, dtype=torch.int32, device=DEV), torch.ones(4, dtype=torch.int32, device=DEV)
    decode = mslk_amd.attention_decode
    refused("GPU", decode, q.cpu(), pool, pool, table, lens)
    refused("one shape", decode, q, pool, pool[:2], table, lens)
    refused("dtype of q", decode, q, pool.half(), pool.half(), table, lens)
    refused("belong to", decode, q, codes, codes, table, lens)
    refused("belong to", decode, q, codes, codes, table, lens, row_scale)
    refused("belong to", decode, q, pool, pool, table, lens, row_scale, row_scale)
    refused("float32 tensors", decode, q, codes, codes, table, lens, row_scale[..., :1], row_scale)
    refused("int32", decode, q, pool, pool, table.long(), lens)
    refused("int32", decode, q, pool, pool, table, lens.cpu())
    refused("one length per row", decode, q, pool, pool, table, lens[:3])
    refused("row per sequence", decode, q, pool, pool, table[:3], lens[:3])
    refused("channels of the cache", decode, q, pool.transpose(2, 3).contiguous().transpose(2, 3), pool, table, lens)
    odd = torch.zeros(3, 16, 2, 68, dtype=torch.bfloat16, device=DEV)[..., :64]
    refused("16-byte boundaries", decode, q, odd, pool, table, lens)
    refused("8-byte boundaries", decode, q, torch.zeros(3, 16, 2, 68, device=DEV).to(F8)[..., :64], codes, table, lens, row_scale, row_scale)
    refused("at least one page", decode, q, pool[:0], pool[:0], table, lens)
    refused("positive", decode, q, pool, pool, table, lens, scale=0.0)

    append = mslk_amd.append_kv
    refused("GPU", append, q.cpu(), k, k, pool, pool, table, lens)
    refused("same tokens", append, q[:3], k, k, pool, pool, table, lens)
    refused("one token per sequence", append, q, k, k, pool, pool, table[:3], lens[:3])
    refused("one offset more", append, q, k, k, pool, pool, table, lens, cu)
    refused("KV heads", append, q, k[:, :1], k[:, :1], pool, pool, table, lens)
    refused("float32 tensor", append, q, k, k, pool, pool, table, lens, rotary=torch.zeros(9, 64, device=DEV).half())
    refused("even in number", append, q, k, k, pool, pool, table, lens, rotary=torch.zeros(9, 63, device=DEV))
    refused("even in number", append, q, k, k, pool, pool, table, lens, rotary=torch.zeros(9, 66, device=DEV))
    refused("at least one position", append, q, k, k, pool, pool, table, lens, rotary=torch.zeros(0, 64, device=DEV))


def test_nothing_joins_a_graph_of_gradients():
    q = torch.randn(4, 2, 64, device=DEV).bfloat16().requires_grad_()
    out = mslk_amd.attention_prompt(q, q, q, offsets([4]).to(DEV))
    assert not out.requires_grad


@pytest.mark.parametrize("fp8", [False, True])
def test_appending_is_seen_as_a_write(fp8):
    """A tensor that was saved for a gradient and then written is refused by the backward pass; tensors made in inference mode, which
    have no version, are written all the same; a compiled step leaves the caches as the eager one does."""
    g = torch.Generator().manual_seed(35)
    rows = heads(g, 2, 8, 64, torch.bfloat16).to(DEV)
    q, k, v = rows[:, :4], rows[:, 4:6], rows[:, 6:]
    table, lens = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV), torch.tensor([3, 20], dtype=torch.int32, device=DEV)

    def caches():
        pools = [torch.zeros(4, 16, 2, 64, device=DEV).to(F8 if fp8 else torch.bfloat16) for _ in range(2)]
        return pools, {"k_scale": torch.zeros(4, 16, 2, device=DEV), "v_scale": torch.zeros(4, 16, 2, device=DEV)} if fp8 else {}

    pools, scales = caches()
    weight = torch.ones(4, 16, 2, 64 if not fp8 else 1, device=DEV, requires_grad=True)
    saved = scales["v_scale"][..., None] if fp8 else pools[1]
    loss = (weight * saved).sum()
    mslk_amd.append_kv(q, k, v, *pools, table, lens, **scales)
    assert all(t._version > 0 for t in (*pools, *scales.values()))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()

    with torch.inference_mode():
        others, other_scales = caches()
    mslk_amd.append_kv(q, k, v, *others, table, lens, **other_scales)
    with torch.inference_mode():
        mslk_amd.append_kv(q, k, v, *others, table, lens, **other_scales)
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip((*pools, *scales.values()), (*others, *other_scales.values())))

    def step(q, k, v, pools, scales):
        turned = mslk_amd.append_kv(q, k, v, *pools, table, lens, **scales)
        return mslk_amd.attention_decode(turned, *pools, table, lens, *scales.values())

    want = step(q, k, v, pools, scales)
    again, again_scales = caches()
    got = torch.compile(step, backend="aot_eager", fullgraph=True)(q, k, v, again, again_scales)
    assert torch.equal(got, want)
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip((*pools, *scales.values()), (*again, *again_scales.values())))


def test_operators_have_shape_functions():
    q, k = torch.randn(4, 4, 64, device=DEV).bfloat16(), torch.randn(4, 2, 64, device=DEV).bfloat16()
    cu = offsets([4]).to(DEV)
    checks = ("test_schema", "test_faketensor")
    torch.library.opcheck(torch.ops.mslk.attention_prompt, (q, k, k, cu), test_utils=checks)
    pools = [torch.randn(3, 16, 2, 64, device=DEV).bfloat16() for _ in range(2)]
    table, lens = torch.zeros(4, 2, dtype=torch.int32, device=DEV), torch.ones(4, dtype=torch.int32, device=DEV)
    torch.library.opcheck(torch.ops.mslk.attention_decode, (q, *pools, table, lens), test_utils=checks)
    torch.library.opcheck(torch.ops.mslk.append_kv, (q, k, k, *pools, torch.tensor([[0], [1], [2], [0]], dtype=torch.int32, device=DEV), lens + torch.tensor(
        [0, 0, 0, 1], dtype=torch.int32, device=DEV)), test_utils=checks)
