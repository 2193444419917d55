"""GPU: the paged entry points where their inputs are out of range, not finite or extreme, and what a failed call leaves."""
import ctypes

import pytest
import torch

from paged_case import U, Case, assert_attention, quantise64

pytestmark = pytest.mark.gpu

import cuda_attn  # noqa: E402

F16, BF16 = torch.float16, torch.bfloat16
STATUS_PAGE = 512
both_kernels = pytest.mark.parametrize("hint", [1, 4096], ids=["rows", "chunk"])


@pytest.fixture(autouse=True)
def _gpu(cuda_ok):
    cuda_attn.device_status()
    yield
    assert cuda_attn.device_status() == 0


def attend(c, causal=True, max_new=0, scale=None):
    return cuda_attn.paged_attn(c.q, *c.where(), **c.scales(), causal=causal, max_new=max_new, scale=scale)


def pools(c):
    return [x for x in (c.k_cache, c.v_cache, c.k_scale, c.v_scale) if x is not None]


def same(x, y):
    """Equal, NaNs in the same places among them."""
    return torch.equal(torch.nan_to_num(x.float(), nan=7.0), torch.nan_to_num(y.float(), nan=7.0))


def soil(shape, dtype):
    """Leaves NaNs in the memory that the next tensor of this size is given."""
    torch.full(shape, float("nan"), device="cuda", dtype=dtype)


# ------------------------------------------------------------------------------------------------ pages out of range


@both_kernels
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype,int8", [(F16, False), (BF16, False), (F16, True), (BF16, True)])
def test_tokens_without_a_page_are_zeros(dtype, int8, d, causal, hint):
    """Within the length, under a page id that is out of range: keys and values of zeros, to the attention (they count in the
    sum of weights) as to paged_read. Single pages, a run of them that covers whole tiles, and all of a sequence's."""
    new, kv = [3, 140, 2, 1], [700, 900, 40, 333]
    c = Case(new, kv, 2, 4, d, 16, dtype, int8)
    bad = [[0, 5, 43], list(range(8, 41)) + [56], [0, 1, 2], [20]]
    for b, pages in enumerate(bad):
        for i, page in enumerate(pages):
            c.table[b, page] = (-1, c.k_cache.shape[0], 1 << 30, -(1 << 31))[i % 4]
            for held in (c.keys, c.values):
                held[b][16 * page:16 * page + 16] = 0
    out = attend(c, causal, hint)
    assert cuda_attn.device_status() == STATUS_PAGE
    assert_attention(out, *c.attention64(causal), dtype, int8)
    assert not out[143:145].any()  # the third sequence has no page at all

    soil((146, 2, d), dtype), soil((146, 2, d), dtype)
    read = cuda_attn.paged_read(*c.where(), 146, dtype=dtype, **c.scales())
    assert cuda_attn.device_status() == STATUS_PAGE
    for got, held in zip(read, (c.keys, c.values)):
        want = torch.cat([x[t - n:] for x, n, t in zip(held, new, kv)])
        assert torch.equal(got, want.to(dtype))

    before = [x.clone() for x in pools(c)]
    x = torch.ones(146, 2, d, device="cuda", dtype=dtype)
    cuda_attn.paged_append(x, x, *c.where(), **c.scales())
    assert cuda_attn.device_status() == STATUS_PAGE
    good = torch.zeros(c.k_cache.shape[0], 16, dtype=torch.bool, device="cuda")
    for b, (n, t) in enumerate(zip(new, kv)):
        for j in range(t - n, t):
            if j // 16 not in bad[b]:
                good[c.table[b, j // 16], j % 16] = True
    q, s = quantise64(x[0, 0])
    for was, now, put in zip(before, pools(c), (q if int8 else x[0, 0], q if int8 else x[0, 0], s, s)):
        was.transpose(1, 2)[good] = put
        assert same(was, now)


@pytest.mark.parametrize("over", [1, 2, 5, 50])
@pytest.mark.parametrize("dtype,int8", [(F16, False), (BF16, True)])
def test_new_tokens_past_the_page_table(dtype, int8, over):
    """kv_lens counts more tokens than the table's row has room for: the new tokens that have a place keep it, those past it
    are not written and read as zeros; a token sees the cached ones before it, as many as there are."""
    new, kv = [5, 140, 1], [160, 320, 320]  # whole pages: 10 and 20 of the table's 20, a length out of range in two rows
    c = Case(new, kv, 2, 4, 128, 16, dtype, int8)
    c.table = c.table[:, :20].contiguous()
    c.lens[1:] += over
    before, x = [p.clone() for p in pools(c)], torch.randn(146, 2, 128, device="cuda", dtype=dtype)
    cuda_attn.paged_append(x, x, *c.where(), **c.scales())
    assert cuda_attn.device_status() == STATUS_PAGE
    packed, at = [], 0
    for b, (n, t) in enumerate(zip(new, c.lens.tolist())):
        for i in range(n):
            j = t - n + i
            if j < (160 if b == 0 else 320):
                packed.append((at + i, int(c.table[b, j // 16]), j % 16))
        at += n
    rows, ids, place = (torch.tensor(y, device="cuda") for y in zip(*packed))
    q, s = quantise64(x[rows])
    for was, put in zip(before, (q, q, s, s) if int8 else (x[rows], x[rows])):
        was[ids, :, place] = put
    assert all(same(was, now) for was, now in zip(before, pools(c)))

    soil((146, 2, 128), dtype), soil((146, 2, 128), dtype)
    k, v = cuda_attn.paged_read(*c.where(), 146, dtype=dtype, **c.scales())
    assert cuda_attn.device_status() == STATUS_PAGE
    want = torch.zeros_like(k)
    want[rows] = (q.float() * s[..., None]).to(dtype) if int8 else x[rows]
    assert torch.equal(k, want) and torch.equal(v, want)

    # the rows of tokens within the room: as with lengths that end there
    for hint in (1, 4096):
        out = attend(c, True, hint)
        assert cuda_attn.device_status() == STATUS_PAGE
        for b, (n, t) in enumerate(zip(new, c.lens.tolist())):
            start = sum(new[:b])
            room = 160 if b == 0 else 320
            inside = max(0, n - max(0, t - room))
            alone = [torch.tensor(y, dtype=torch.int32, device="cuda") for y in ([min(t, room)], [0, n])]
            ask = c.q[start:start + n]
            every = cuda_attn.paged_attn(ask, c.k_cache, c.v_cache, c.table[b:b + 1], *alone, **c.scales(), causal=False, max_new=hint)
            past = torch.arange(n, device="cuda") >= inside
            tol = 2.0 ** -7 if dtype == BF16 else 2.0 ** -10  # two sums of the same terms, rounded to 16 bits each
            assert ((out[start:start + n] - every).abs()[past] <= tol * (1 + every.abs()[past])).all()
            if inside:
                alone[0][0], alone[1][1] = min(t, room), inside
                some = cuda_attn.paged_attn(ask[:inside], c.k_cache, c.v_cache, c.table[b:b + 1], *alone, **c.scales(), max_new=hint)
                diff = (out[start:start + inside] - some).abs()
                assert (diff <= tol * (1 + some.abs())).all()
    cuda_attn.device_status()


# ------------------------------------------------------------------------------------------------ packed rows of no sequence


@both_kernels
@pytest.mark.parametrize("lead,trail", [(1, 0), (3, 4), (700, 5), (0, 900)])
@pytest.mark.parametrize("d,int8", [(64, False), (128, True)])
def test_packed_tokens_before_and_after_the_sequences(d, int8, lead, trail, hint):
    """cu_new of a slice: tokens before its first are of no sequence, which is out of range; those after its last may be."""
    c = Case([2, 40, 3], [50, 60, 500], 3, 4, d, 16, F16, int8)
    want = attend(c, True, hint)
    n = c.total
    c.cu += lead
    q = torch.ones(lead + n + trail, 12, d, device="cuda", dtype=F16)
    q[lead:lead + n] = c.q
    for _ in range(2):
        soil(q.shape, F16)
        out = cuda_attn.paged_attn(q, *c.where(), **c.scales(), max_new=hint)
        assert cuda_attn.device_status() == (STATUS_PAGE if lead else 0)
        assert torch.equal(out[lead:lead + n], want)
        assert not out[:lead].any() and not out[lead + n:].any()
    soil((lead + n + trail, 3, d), F16), soil((lead + n + trail, 3, d), F16)
    k, v = cuda_attn.paged_read(*c.where(), lead + n + trail, dtype=F16, **c.scales())
    assert cuda_attn.device_status() == (STATUS_PAGE if lead else 0)
    for x in (k, v):
        assert not x[:lead].any() and not x[lead + n:].any()
    before = [x.clone() for x in pools(c)]
    x = torch.zeros(lead + n + trail, 3, d, device="cuda", dtype=F16)
    x[:lead] = x[lead + n:] = 1.0
    x[lead:lead + n] = k[lead:lead + n]
    cuda_attn.paged_append(x, x, *c.where(), **c.scales())
    assert cuda_attn.device_status() == (STATUS_PAGE if lead else 0)
    if not int8:
        assert same(before[0], c.k_cache)  # the new tokens' own keys were written, and nothing else


# ------------------------------------------------------------------------------------------------ values that are not finite


@both_kernels
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_nan_of_a_16_bit_key_reaches_the_rows_that_see_it(dtype, d, hint):
    """At every place of a stretch of keys, the causal edge among them; no other row changes."""
    c = Case([5], [300], 2, 2, d, 16, dtype, False)
    clean = attend(c, True, hint)
    ids, place = c.places(0, 300)
    for j in list(range(0, 300, 37)) + list(range(262, 300)):
        at = (ids[j], 0, place[j], j % d)
        was = c.k_cache[at].clone()
        c.k_cache[at] = float("nan")
        out = attend(c, True, hint)
        sees = max(0, j - 295)  # the first row that does
        assert out[sees:, :2].isnan().all(), j
        assert torch.equal(out[:sees], clean[:sees]) and torch.equal(out[:, 2:], clean[:, 2:]), j
        c.k_cache[at] = was


@both_kernels
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_infinite_keys(dtype, hint):
    """An infinite key gives an infinite score: NaN where it is positive, no weight where it is negative. In the first tile
    of a row and in a later one."""
    for j in list(range(3, 19)) + list(range(250, 266)):
        c = Case([4], [300], 1, 8, 128, 16, dtype, False)
        ids, place = c.places(0, 300)
        c.k_cache[ids[j], 0, place[j], 5] = c.keys[0][j, 0, 5] = float("inf")
        c.q[..., 5] = torch.where(c.q[..., 5].abs() < 0.25, 0.25, c.q[..., 5])
        out = attend(c, True, hint)
        ref, size = c.attention64(True)
        up = c.q[..., 5] > 0
        assert out[up].isnan().all(), j
        assert_attention(out[~up], ref[~up], size[~up], dtype)


@both_kernels
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype,int8,huge", [(F16, False, 6e4), (BF16, False, 3e38), (BF16, True, 3e38)])
def test_hidden_values_of_any_size_have_no_weight(dtype, int8, huge, d, hint):
    """The last 60 new tokens' values are the largest finite numbers; the rows before do not see them."""
    c = Case([200, 130], [200, 700], 2, 2, d, 16, dtype, int8)
    clean = attend(c, True, hint)
    for b, t in enumerate(c.kv):
        ids, place = (x[t - 60:] for x in c.places(b, t))
        if int8:
            c.v_scale[ids, :, place] = huge / 127
        else:
            c.v_cache[ids, :, place] = huge
    out = attend(c, True, hint)
    for rows in (slice(0, 140), slice(200, 270)):
        assert torch.equal(out[rows], clean[rows])


@both_kernels
@pytest.mark.parametrize("int8", [False, True])
def test_large_scores_stay_between_the_values(int8, hint):
    """Scores in the hundreds: a softmax of one or two keys, which none of an output's columns leaves: beyond the least and the
    largest value that its row sees lies only what rounding the probabilities and the output moves it by (paged_case)."""
    c = Case([3, 200], [700, 300], 2, 2, 128, 16, BF16, int8, scale=8.0)
    c.q.mul_(8.0)
    out = attend(c, True, hint).double()
    at = 0
    for b, (n, t) in enumerate(zip(c.new, c.kv)):
        v = c.values[b]
        lo, hi, size = (f(0)[0][t - n:].repeat_interleave(2, 1) for f in (v.cummin, v.cummax, v.abs().cummax))
        tol = (U[BF16] + 2 * (2.0 ** -11 if int8 else U[BF16]) + 2.0 ** -12) * size
        o = out[at:at + n]
        assert ((o >= lo - tol) & (o <= hi + tol)).all()
        at += n


@both_kernels
@pytest.mark.parametrize("dtype,int8", [(F16, False), (BF16, False), (BF16, True)])
def test_a_scale_of_next_to_nothing(dtype, int8, hint):
    """The least scales that float32 holds: every key that a row sees has the same weight."""
    c = Case([2, 130], [300, 200], 1, 4, 64, 16, dtype, int8)
    assert_attention(attend(c, True, hint, 1e-40), *c.attention64(True, 0.0), dtype, int8)


# ------------------------------------------------------------------------------------------------ after a wait that gave up


def test_the_status_names_all_that_happened(capi):
    """A wait that gave up does not hide that a page was out of range too, nor the reverse."""
    status = ctypes.c_int()
    c = Case([1], [40], 1, 1, 64, 16, F16, False)
    c.table.fill_(-1)
    for probe, page in ((False, True), (True, True)):
        if page:
            attend(c)
        if probe:
            capi.wait_expiry_probe()
        assert capi.lib.phantom_attn_device_status(ctypes.byref(status)) != 0
        said = capi.last_error()
        assert ("wait expired" in said) == probe and ("out of range" in said) == page, said


def test_a_replay_after_one_that_gave_up():
    """A captured call whose length grows to 6e8 tokens (all in one page) keeps a CTA at its part for longer than a wait's
    limit of a second: the call ends soon after and says so. The counts of the parts that were done must not stay for the
    next replays, which would join parts that are not there yet."""
    heads, page, small, huge = 60, 1024, 1 << 16, 617 << 20
    kc, vc = (torch.randn(1, heads, page, 128, device="cuda").to(BF16) for _ in "kv")
    table = torch.zeros(1, 617 << 10, dtype=torch.int32, device="cuda")
    lens = torch.tensor([small], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    q = torch.randn(1, heads, 128, device="cuda").to(BF16)

    def step():
        return cuda_attn.paged_attn(q, kc, vc, table, lens, cu, max_new=1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step()

    def replays(n):
        wrong = 0
        for _ in range(n):
            q.copy_(torch.randn(1, heads, 128, device="cuda"))
            graph.replay()
            got = o.clone()
            wrong += not torch.equal(got, step())
        return wrong

    assert replays(20) == 0
    lens.fill_(huge)
    graph.replay()
    status = cuda_attn.device_status()
    assert status & 15 and not status & STATUS_PAGE
    lens.fill_(small)
    assert replays(40) == 0
    del graph
