"""GPU: the paged key/value cache (append, read back) and the attention over it, against their definitions in 64 bits."""
import ctypes
import random

import pytest
import torch

from paged_case import U, Case, assert_attention, quantise64

pytestmark = pytest.mark.gpu

import cuda_attn  # noqa: E402

F16, BF16 = torch.float16, torch.bfloat16
STATUS_PAGE = 512


@pytest.fixture(autouse=True)
def _gpu(cuda_ok):
    cuda_attn.device_status()
    yield
    assert cuda_attn.device_status() == 0


def attend(c, causal=True, max_new=0, scale=None):
    return cuda_attn.paged_attn(c.q, *c.where(), **c.scales(), causal=causal, max_new=max_new, scale=scale)


def check(c, causal=True, max_new=0, scale=None):
    out = attend(c, causal, max_new, scale)
    assert out.shape == c.q.shape and out.dtype == c.dtype and out.is_contiguous()
    assert_attention(out, *c.attention64(causal, scale), c.dtype, c.int8)
    return out


# new and cached tokens: single tokens at every place of a tile's and a page's edge; few and many; none; more than cached
LENGTHS = {
    "tokens": ([1] * 11, [1, 2, 16, 17, 63, 64, 65, 127, 128, 129, 1000]),
    "absent": ([1, 0, 1, 0, 1], [70, 0, 0, 40, 300]),
    "few": ([3, 1, 5, 2], [3, 200, 77, 130]),
    "chunks": ([130, 0, 1, 257, 33], [130, 5, 900, 700, 1025]),
    "rows_without_keys": ([5, 300, 2], [3, 100, 0]),
}


@pytest.mark.parametrize("hint", [1, 4096], ids=["rows", "chunk"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths", list(LENGTHS))
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype,int8", [(F16, False), (BF16, False), (F16, True), (BF16, True)])
def test_attention(dtype, int8, d, lengths, causal, hint):
    new, kv = LENGTHS[lengths]
    check(Case(new, kv, 2, 4, d, 16, dtype, int8), causal, hint)


@pytest.mark.parametrize("hint", [1, 4096], ids=["rows", "chunk"])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("group,heads", [(1, 3), (2, 2), (3, 2), (5, 1), (7, 1), (8, 2), (16, 1), (20, 1), (48, 1), (128, 1)])
def test_attention_shared_heads(group, heads, int8, hint):
    check(Case([1, 40, 7], [500, 40, 333], heads, group, 128, 32, BF16, int8), True, hint)


@pytest.mark.parametrize("hint", [1, 4096], ids=["rows", "chunk"])
@pytest.mark.parametrize("layout", ["plain", "interleaved", "token"])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("int8", [False, True])
def test_attention_pages_and_strides(page, layout, int8, hint):
    c = Case([1, 150, 20], [1500, 700, 257], 2, 2, 64, page, F16, int8, layout=layout)
    check(c, True, hint)


@pytest.mark.parametrize("hint", [1, 4096], ids=["rows", "chunk"])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("stale", [float("nan"), float("inf"), -3e4])
def test_attention_ignores_what_lies_past_the_length(stale, int8, hint):
    check(Case([1, 3, 140], [33, 100, 150], 2, 4, 128, 64, F16, int8, stale=stale), True, hint)


@pytest.mark.parametrize("hint", [1, 4096], ids=["rows", "chunk"])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_of_many_sequences(dtype, int8, hint):
    """More sequences than a warp has lanes; long and short mixed, several CTAs to one sequence and the reverse."""
    rng = random.Random(5)
    kv = [rng.choice([1, 7, 100, 400, 3500]) for _ in range(75)]
    check(Case([min(t, rng.choice([0, 1, 1, 2])) for t in kv], kv, 2, 4, 128, 16, dtype, int8), True, hint)


@pytest.mark.parametrize("hint", [1, 4096], ids=["rows", "chunk"])
@pytest.mark.parametrize("dtype,int8", [(F16, False), (BF16, True)])
def test_one_long_sequence_is_shared(dtype, int8, hint):
    check(Case([1], [40000], 1, 8, 128, 128, dtype, int8), True, hint)


@pytest.mark.parametrize("hint", [1, 4096], ids=["rows", "chunk"])
@pytest.mark.parametrize("scale", [0.02, -0.05, 0.5])
def test_attention_scale(scale, hint):
    check(Case([2, 130], [300, 200], 1, 4, 64, 16, F16, False), True, hint, scale)


@pytest.mark.parametrize("hint", [1, 4096], ids=["rows", "chunk"])
@pytest.mark.parametrize("int8", [False, True])
def test_large_scores(int8, hint):
    """Scores in the hundreds: a softmax of one or two keys. What the scores' fp32 rounding moves the weights by is 128
    2^-24 of sums of products near 1e4, too much for the bound of ordinary scores only in rows whose two best are close, so
    the outputs are held to lie between the values' extremes and the norm of the error to a hundredth."""
    c = Case([3, 200], [700, 300], 2, 2, 128, 16, BF16, int8, scale=8.0)
    c.q.mul_(8.0)
    out = attend(c, True, hint)
    ref, _ = c.attention64(True)
    assert torch.isfinite(out).all()
    assert (out.double() - ref).norm() <= 1e-2 * ref.norm()


@pytest.mark.parametrize("hint", [1, 4096], ids=["rows", "chunk"])
@pytest.mark.parametrize("dtype,power", [(BF16, 60), (BF16, -60), (F16, -12)])
@pytest.mark.parametrize("int8", [False, True])
def test_values_far_from_one(dtype, power, int8, hint):
    """Values of 2^power: the probabilities' 16-bit form must not depend on the values' size."""
    c = Case([2, 100], [300, 150], 1, 4, 64, 16, dtype, int8)
    x = 2.0 ** power
    if int8:
        c.v_scale.mul_(x)
    else:
        c.v_cache.mul_(x)
    c.values = [v * x for v in c.values]
    out = attend(c, True, hint)
    ref, size = c.attention64(True)
    u = U[dtype]
    bound = u * ref.abs() + (2 * u + 2.0 ** -12) * size + (2.0 ** -24 if dtype == F16 else 0.0)
    assert ((out.double() - ref).abs() <= bound).all()


def test_vectors_of_very_different_scales():
    """8-bit values whose scales span 2^-20 to 2^20 within one sequence, zeros among them."""
    c = Case([4], [600], 1, 4, 128, 16, BF16, True, seed=3)
    ids, place = c.places(0, 600)
    f = torch.exp2(torch.randint(-20, 21, (600, 1), device="cuda").float())
    f[::7] = 2.0 ** -100 / c.v_scale[ids, :, place][::7].clamp_min(1e-30)
    c.v_scale[ids, :, place] *= f
    c.values[0] = c.v_cache[ids, :, place].double() * c.v_scale[ids, :, place].double()[..., None]
    for hint in (1, 4096):
        check(c, True, hint)


@pytest.mark.parametrize("hint", [1, 4096], ids=["rows", "chunk"])
def test_zero_scales_and_zero_queries(hint):
    """8-bit caches of other writers: vectors of zeros with the scale 0 count in the sum of weights; and queries of zeros or
    of very different sizes."""
    c = Case([3], [500], 1, 4, 64, 16, BF16, True, seed=4)
    ids, place = c.places(0, 500)
    for cache, scale, held in ((c.k_cache, c.k_scale, c.keys), (c.v_cache, c.v_scale, c.values)):
        cache[ids[::5], :, place[::5]] = 0
        scale[ids[::5], :, place[::5]] = 0.0
        held[0][::5] = 0.0
    c.q[0, 1] = 0
    c.q[1] *= 2.0 ** -100
    c.q[2, 2, 7] = 300.0
    check(c, True, hint)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new,group,hint", [([1, 1, 1], 16, 1), ([2, 0, 2], 12, 2), ([5, 1, 3], 9, 1), ([1, 2, 1], 16, 2)])
@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 128), (BF16, 64), (F16, 64)])
def test_long_8_bit_contexts_of_9_to_32_rows(dtype, d, new, group, hint, causal):
    """Units of 16 rows: taken where the keys of 4 heads and 3 sequences with room for 10240 tokens are read more than once."""
    check(Case(new, [8000, 500, 3333], 4, group, d, 1024, dtype, True), causal, hint)


@pytest.mark.parametrize("dtype,int8", [(BF16, False), (BF16, True), (F16, False)])
@pytest.mark.parametrize("new", [[3] * 4, [8, 1, 0, 5]])
def test_a_few_new_tokens(new, dtype, int8):
    """Several blocks of rows to a sequence, as many as max_new says."""
    check(Case(new, [700, 33, 64, 300], 2, 4, 128, 16, dtype, int8), True, max(new))


@pytest.mark.parametrize("hint", [1, 4096], ids=["rows", "chunk"])
def test_only_rows_that_see_a_nan_turn_nan(hint):
    """8-bit caches: a vector with a NaN was appended as the last but one of the new tokens."""
    for scales in ("k_scale", "v_scale"):
        c = Case([5], [300], 2, 2, 128, 16, F16, True)
        clean = attend(c, True, hint)
        ids, place = c.places(0, 300)
        getattr(c, scales)[ids[298], 0, place[298]] = float("nan")
        out = attend(c, True, hint)
        assert out[3:, :2].isnan().all()
        assert torch.equal(out[:3], clean[:3]) and torch.equal(out[:, 2:], clean[:, 2:])


def test_results_repeat_bit_for_bit():
    for int8 in (False, True):
        for hint in (1, 4096):
            c = Case([1, 60, 2], [5000, 600, 90], 2, 4, 128, 16, BF16, int8)
            first = attend(c, True, hint)
            for _ in range(3):
                assert torch.equal(attend(c, True, hint), first)


def test_graph_replay_follows_the_lengths():
    """A captured step, replayed as kv_lens and the page table change on the device."""
    c = Case([1, 1, 1], [900, 300, 40], 2, 4, 128, 16, BF16, False)
    k, v = (torch.randn(3, 2, 128, device="cuda").to(BF16) for _ in "kv")
    saved = c.lens.clone()

    def step():
        cuda_attn.paged_append(k, v, *c.where())
        return cuda_attn.paged_attn(c.q, *c.where(), max_new=1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step()
    for shrink in (0, 3, 17):
        c.lens.copy_(saved - shrink)
        graph.replay()
        got = o.clone()
        assert torch.equal(got, step())
    del graph


def test_calls_on_streams_of_their_own():
    cases = [Case([1, 30], [2000 + 300 * i, 500], 2, 4, 64, 16, F16, i % 2 == 1, seed=i) for i in range(4)]
    want = [attend(c, True, h) for c in cases for h in (1, 4096)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for c, s in zip(cases, streams):
        with torch.cuda.stream(s):
            got += [attend(c, True, h) for h in (1, 4096)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_packed_tokens_of_no_sequence_get_zeros():
    c = Case([2, 3], [50, 60], 1, 4, 64, 16, F16, False)
    q = torch.cat([c.q, torch.ones(4, 4, 64, device="cuda", dtype=F16)])
    for hint in (1, 4096):
        out = cuda_attn.paged_attn(q, *c.where(), max_new=hint)
        cuda_attn.device_status()
        assert torch.equal(out[:5], attend(c, True, hint)) and not out[5:].any()


# ------------------------------------------------------------------------------------------------ append and read


@pytest.mark.parametrize("layout", ["plain", "interleaved", "token"])
@pytest.mark.parametrize("heads,d", [(1, 64), (3, 128), (8, 128), (16, 64)])
@pytest.mark.parametrize("dtype,int8", [(F16, False), (BF16, False), (F16, True), (BF16, True)])
def test_append_then_read(dtype, int8, heads, d, layout):
    """What append writes is what the definition says, whole numbers and scales exactly; nothing else changes; read gives
    the products rounded once."""
    new, kv = [1, 40, 0, 17, 300], [1, 100, 20, 17, 1000]
    c = Case(new, kv, heads, 1, d, 32, dtype, int8, layout=layout)
    g = torch.Generator(device="cuda").manual_seed(9)
    wide = torch.randn(c.total, 2 * heads + 1, d, device="cuda", generator=g).to(dtype)
    k, v = wide[:, 1:heads + 1], wide[:, heads + 1:]
    k[0, 0] = 0
    k[1, 0] *= 2.0 ** -20 if dtype == BF16 else 2.0 ** -3
    v[2, -1] = 1.0
    v[2, -1, 3:9] = 0.5  # 63.5: a tie
    before = [x.clone() for x in (c.k_cache, c.v_cache)] + ([c.k_scale.clone(), c.v_scale.clone()] if int8 else [])
    cuda_attn.paged_append(k, v, *c.where(), **c.scales())
    rk, rv = cuda_attn.paged_read(*c.where(), c.total, dtype=dtype, **c.scales())
    at = 0
    for b, (n, t) in enumerate(zip(new, kv)):
        ids, place = c.places(b, t)
        ids, place = ids[t - n:], place[t - n:]
        for j, (x, cache, sc, back) in enumerate(((k, c.k_cache, c.k_scale, rk), (v, c.v_cache, c.v_scale, rv))):
            x, back = x[at:at + n], back[at:at + n]
            if int8:
                q, s = quantise64(x)
                assert torch.equal(cache[ids, :, place], q)
                assert torch.equal(sc[ids, :, place], s)
                assert torch.equal(back, (q.float() * s[..., None]).to(dtype))
                before[2 + j][ids, :, place] = s
                before[j][ids, :, place] = q
            else:
                assert torch.equal(cache[ids, :, place], x) and torch.equal(back, x)
                before[j][ids, :, place] = x
        at += n
    for x, y in zip(before, [c.k_cache, c.v_cache] + ([c.k_scale, c.v_scale] if int8 else [])):
        assert torch.equal(torch.nan_to_num(x, nan=7.0) if x.is_floating_point() else x,
                           torch.nan_to_num(y, nan=7.0) if y.is_floating_point() else y)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_quantisation_over_all_magnitudes(dtype):
    """Every 16-bit pattern of a vector against many largest values: the whole numbers are those of exact arithmetic."""
    bits = torch.randint(0, 1 << 16, (4096, 4, 128), device="cuda", dtype=torch.int32, generator=torch.Generator("cuda").manual_seed(1))
    x = bits.to(torch.int16).view(dtype)
    x = torch.where(torch.isfinite(x), x, 1.0).to(dtype)
    keep = torch.rand(4096, 4, 1, device="cuda") < 0.5  # half of the vectors: values of similar size, where ties are
    x = torch.where(keep, (torch.randint(-255, 256, x.shape, device="cuda").to(dtype) / 64), x)
    c = Case([4096], [4096], 4, 1, 128, 64, dtype, True)
    cuda_attn.paged_append(x, x, *c.where(), **c.scales())
    ids, place = c.places(0, 4096)
    q, s = quantise64(x)
    assert torch.equal(c.k_cache[ids, :, place], q) and torch.equal(c.v_scale[ids, :, place], s)


def test_non_finite_vectors_read_back_as_nan():
    c = Case([4], [4], 2, 1, 64, 16, F16, True)
    x = torch.randn(4, 2, 64, device="cuda").to(F16)
    x[1, 0, 5], x[2, 1, 63], x[3, 0, 0] = float("inf"), float("nan"), float("-inf")
    cuda_attn.paged_append(x, x, *c.where(), **c.scales())
    k, v = cuda_attn.paged_read(*c.where(), 4, dtype=F16, **c.scales())
    for y in (k, v):
        for t, h in ((1, 0), (2, 1), (3, 0)):
            assert y[t, h].isnan().all()
        assert torch.isfinite(y[0]).all() and torch.isfinite(y[1, 1]).all() and torch.isfinite(y[2, 0]).all()


@pytest.mark.parametrize("int8", [False, True])
def test_offsets_past_32_bits(int8):
    """A pool of more than 2^32 bytes: the last pages are reached, by every operator."""
    page, d, pages = 128, 128, (1 << 32) // (128 * 128) + 700 if int8 else (1 << 31) // (128 * 128) + 700
    kc = torch.empty(pages, 1, page, d, device="cuda", dtype=torch.int8 if int8 else F16)
    vc = torch.empty_like(kc)
    sc = {"k_scale": None, "v_scale": None}
    if int8:
        sc = {n: torch.empty(pages, 1, page, device="cuda") for n in sc}
    n = 300
    table = torch.tensor([[pages - 1, 0, pages - 3, -1]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    k, v = (torch.randn(n, 1, d, device="cuda").to(F16) for _ in "kv")
    cuda_attn.paged_append(k, v, kc, vc, table, lens, cu, **sc)
    rk, rv = cuda_attn.paged_read(kc, vc, table, lens, cu, n, dtype=F16, **sc)
    tol = 0.006 if int8 else 0.0  # half a step of max|x| / 127, and its rounding
    assert (rk.float() - k.float()).abs().max() <= tol * k.abs().max() and (rv.float() - v.float()).abs().max() <= tol * v.abs().max()
    q = torch.randn(n, 4, d, device="cuda").to(F16)
    for hint in (1, 4096):
        o = cuda_attn.paged_attn(q, kc, vc, table, lens, cu, **sc, max_new=hint)
        s = (q.double().transpose(0, 1) @ rk.double()[:, 0].T) / d ** 0.5
        s = s.masked_fill(torch.ones(n, n, device="cuda").triu(1).bool(), -torch.inf).softmax(-1)
        ref = (s @ rv.double()[:, 0]).transpose(0, 1)
        assert (o.double() - ref).norm() <= 1e-3 * ref.norm()


# ------------------------------------------------------------------------------------------------ out of range, refusals


@pytest.mark.parametrize("int8", [False, True])
def test_out_of_range_is_not_followed(int8):
    """Page ids, lengths and offsets that the kernels bound: the call ends, says so, and leaves the pool alone."""
    c = Case([1, 40], [100, 90], 2, 4, 64, 16, F16, int8)
    k = torch.ones(41, 2, 64, device="cuda", dtype=F16)

    def all_three():
        cuda_attn.paged_append(k, k, *c.where(), **c.scales())
        cuda_attn.paged_read(*c.where(), 41, dtype=F16, **c.scales())
        for hint in (1, 4096):
            attend(c, True, hint)
        return cuda_attn.device_status()

    assert all_three() == 0
    for broken in ("page", "negative", "length", "offset"):
        table, lens, cu = c.table.clone(), c.lens.clone(), c.cu.clone()
        pool = c.k_cache.clone()
        if broken == "page":
            c.table[0, 6] = 1 << 30
            c.table[1, 2] = c.k_cache.shape[0]
        elif broken == "negative":
            c.table.fill_(-5)
        elif broken == "length":
            c.lens[0], c.lens[1] = 1 << 30, -4
        else:
            c.cu[1], c.cu[2] = -7, 1 << 29
        assert all_three() == STATUS_PAGE
        if broken == "negative":
            assert torch.equal(torch.nan_to_num(pool), torch.nan_to_num(c.k_cache))
        c.table.copy_(table), c.lens.copy_(lens), c.cu.copy_(cu)
        assert all_three() == 0


def test_refusals():
    c = Case([1, 2], [20, 30], 2, 4, 64, 16, F16, False)
    i = Case([1, 2], [20, 30], 2, 4, 64, 16, F16, True)
    kc, vc, table, lens, cu = c.where()
    k = torch.zeros(3, 2, 64, device="cuda", dtype=F16)
    attn = cuda_attn.paged_attn
    for match, call in [
        ("float16 or bfloat16", lambda: attn(c.q.float(), *c.where())),
        ("dtype", lambda: attn(c.q.bfloat16(), *c.where())),
        ("CUDA tensors", lambda: attn(c.q.cpu(), *c.where())),
        ("CUDA tensors", lambda: attn(c.q, kc, vc, table.cpu(), lens, cu)),
        ("int32", lambda: attn(c.q, kc, vc, table.long(), lens, cu)),
        ("batch", lambda: attn(c.q, kc, vc, table, lens, cu[:2])),
        ("k_scale and v_scale", lambda: attn(i.q, *i.where())),
        ("k_scale and v_scale", lambda: attn(c.q, *c.where(), **i.scales())),
        ("scales must be", lambda: attn(i.q, *i.where(), k_scale=i.k_scale.half(), v_scale=i.v_scale)),
        ("query heads", lambda: attn(c.q[:, :3], *c.where())),
        ("cache's d", lambda: attn(torch.zeros(3, 8, 128, device="cuda", dtype=F16), *c.where())),
        ("head dimension", lambda: attn(c.q[..., :32], kc[..., :32], vc[..., :32], table, lens, cu)),
        ("page size", lambda: attn(c.q, kc[:, :, :8], vc[:, :, :8], table, lens, cu)),
        ("page size", lambda: attn(c.q, kc.repeat(1, 1, 3, 1), vc.repeat(1, 1, 3, 1), table, lens, cu)),
        ("contiguous", lambda: attn(torch.zeros(3, 8, 128, device="cuda", dtype=F16)[..., ::2], *c.where())),
        ("16 bytes", lambda: attn(torch.zeros(3, 8, 68, device="cuda", dtype=F16)[..., :64], *c.where())),
        ("16-byte aligned", lambda: attn(torch.zeros(3 * 8 * 64 + 4, device="cuda", dtype=F16)[4:].view(3, 8, 64), *c.where())),
        ("scale must be finite", lambda: attn(c.q, *c.where(), scale=float("nan"))),
        ("scale must be finite", lambda: attn(c.q, *c.where(), scale=0.0)),
        ("max_new", lambda: attn(c.q, *c.where(), max_new=-1)),
        ("must have", lambda: cuda_attn.paged_append(k, k[:, :1], *c.where())),
        ("heads", lambda: cuda_attn.paged_append(k[:, :1], k[:, :1], *c.where())),
        ("dtype", lambda: cuda_attn.paged_append(k.bfloat16(), k.bfloat16(), *c.where())),
        ("dtype", lambda: cuda_attn.paged_read(*i.where(), 3, dtype=torch.float32, **i.scales())),
        ("total", lambda: cuda_attn.paged_read(*c.where(), -1)),
    ]:
        with pytest.raises(RuntimeError, match=match):
            call()


def test_nothing_to_do():
    c = Case([0, 0], [20, 0], 2, 4, 64, 16, F16, False)
    assert attend(c).shape == (0, 8, 64)
    k, v = cuda_attn.paged_read(*c.where(), 0)
    assert k.shape == v.shape == (0, 2, 64)
    cuda_attn.paged_append(k, v, *c.where())


def test_c_abi(capi):
    """The three entry points of the C ABI through ctypes."""
    from cuda_attn.capi import BF16 as C_BF16, I8, PagedCache
    c = Case([1, 20], [300, 45], 2, 4, 128, 16, BF16, True)
    p = PagedCache(c.k_cache.data_ptr(), c.v_cache.data_ptr(), c.k_scale.data_ptr(), c.v_scale.data_ptr(),
                   c.k_cache.stride()[:3], c.v_cache.stride()[:3], c.k_scale.stride()[:2], c.v_scale.stride()[:2],
                   c.table.data_ptr(), c.lens.data_ptr(), c.cu.data_ptr(), 2, c.table.shape[1], c.table.stride(0),
                   c.k_cache.shape[0], 16, 2, 128, I8)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    o, k, v = torch.empty_like(c.q), *(torch.empty(21, 2, 128, device="cuda", dtype=BF16) for _ in "kv")
    capi._check(capi.lib.phantom_attn_paged(p, c.q.data_ptr(), c.q.stride(0), c.q.stride(1), o.data_ptr(), 21, 8, C_BF16, 1, 0.0, 0, stream))
    capi._check(capi.lib.phantom_attn_paged_read(p, k.data_ptr(), v.data_ptr(), 21, C_BF16, stream))
    assert torch.equal(o, attend(c))
    rk, rv = cuda_attn.paged_read(*c.where(), 21, **c.scales())
    assert torch.equal(k, rk) and torch.equal(v, rv)
    capi._check(capi.lib.phantom_attn_paged_append(p, k.data_ptr(), v.data_ptr(), 256, 128, 256, 128, 21, C_BF16, stream))
    rk2, _ = cuda_attn.paged_read(*c.where(), 21, **c.scales())
    assert (rk2.float() - rk.float()).abs().max() <= 0.006 * rk.float().abs().max()
    capi.launch_count(reset=True)
    assert capi.lib.phantom_attn_paged(None, None, 0, 0, None, 1, 1, C_BF16, 1, 0.0, 0, stream) != 0 and "null cache" in capi.last_error()
    assert capi.launch_count() == 0


@pytest.mark.parametrize("int8,dtype", [(False, BF16), (True, BF16), (True, F16)])
def test_serving_example(int8, dtype):
    """Prompts in chunks and decoding over reused pages; every finished sequence against the dense fp32 kernel on the
    tokens read back: they differ by the output's rounding, the probabilities', and, for int8, the read back tokens'."""
    from cuda_attn import serve_paged
    server, worst, steps = serve_paged.run(8, pages=150, chunk=200, int8=int8, dtype=dtype, d=64, heads=2)
    assert worst <= (8e-3 if dtype == BF16 else 1e-3) and steps > 40 and len(server.pool.free) == 150
