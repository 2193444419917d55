"""CPU: what the paged entry points refuse before they touch a GPU, and the serving example's page bookkeeping."""
import ctypes

import pytest
import torch

import cuda_attn
from cuda_attn.capi import BF16, ERR_INVALID, ERR_UNSUPPORTED, F16, F32, I8, CAPI, PagedCache


@pytest.fixture(scope="module")
def lib():
    return CAPI()


def cache(**kw):
    """A well-formed descriptor (its pointers are never followed: the checks below come first)."""
    c = PagedCache(4096, 4096, None, None, (2048, 1024, 64), (2048, 1024, 64), (0, 0), (0, 0), 4096, 4096, 4096, 2, 8, 8, 32, 16, 2, 64, F16)
    for name, value in kw.items():
        setattr(c, name, value)
    return c


def calls(lib, c, total=3, dtype=F16):
    yield lib.lib.phantom_attn_paged_append(c, 4096, 4096, 128, 64, 128, 64, total, dtype, None)
    yield lib.lib.phantom_attn_paged_read(c, 4096, 4096, total, dtype, None)
    yield lib.lib.phantom_attn_paged(c, 4096, 512, 64, 4096, total, 8, dtype, 1, 0.0, 0, None)


@pytest.mark.parametrize("what,code,text", [
    (dict(batch=0), ERR_INVALID, "non-empty"),
    (dict(heads=0), ERR_INVALID, "non-empty"),
    (dict(num_pages=-1), ERR_INVALID, "non-empty"),
    (dict(table_width=0), ERR_INVALID, "non-empty"),
    (dict(head_dim=96), ERR_UNSUPPORTED, "head dimension"),
    (dict(dtype=BF16), ERR_INVALID, "dtype"),
    (dict(dtype=F32), ERR_INVALID, "dtype"),
    (dict(page_size=8), ERR_UNSUPPORTED, "page size"),
    (dict(page_size=48), ERR_UNSUPPORTED, "page size"),
    (dict(page_size=2048), ERR_UNSUPPORTED, "page size"),
    (dict(batch=70000), ERR_UNSUPPORTED, "65535"),
    (dict(table_stride=7), ERR_INVALID, "overlap"),
    (dict(k_stride=(2048, 1024, 60)), ERR_INVALID, "16 bytes"),
    (dict(v_stride=(-2048, 1024, 64)), ERR_INVALID, "16 bytes"),
    (dict(k_stride=(1 << 40, 1024, 64)), ERR_INVALID, "16 bytes"),
    (dict(dtype=I8, k_scale_stride=(18, 16)), ERR_INVALID, "scale strides"),
])
def test_refusals(lib, what, code, text):
    for rc in calls(lib, cache(**what)):
        assert rc == code and text in lib.last_error(), (rc, lib.last_error())


def test_refusals_of_the_packed_arrays(lib):
    for rc in calls(lib, cache(), total=0):
        assert rc == ERR_INVALID and "non-empty" in lib.last_error()
    for rc in calls(lib, cache(), dtype=F32):
        assert rc == ERR_UNSUPPORTED and "float16" in lib.last_error()
    for rc in calls(lib, None):
        assert rc == ERR_INVALID and "null cache" in lib.last_error()


def test_descriptor_matches_the_header():
    """The ctypes structure has the C structure's size and offsets (natural alignment, as declared)."""
    assert PagedCache.k_stride.offset == 32 and PagedCache.page_table.offset == 112 and PagedCache.batch.offset == 136
    assert ctypes.sizeof(PagedCache) == 168 and PagedCache.dtype.offset == 164


def test_torch_binding_rejects_cpu_tensors():
    kc = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    i = torch.zeros(1, 2, dtype=torch.int32)
    q = torch.zeros(1, 4, 64, dtype=torch.float16)
    for call in (lambda: cuda_attn.paged_attn(q, kc, kc, i, i[0, :1], i[0]), lambda: cuda_attn.paged_read(kc, kc, i, i[0, :1], i[0], 1),
                 lambda: cuda_attn.paged_append(q[:, :2], q[:, :2], kc, kc, i, i[0, :1], i[0])):
        with pytest.raises(RuntimeError, match="CUDA tensors"):
            call()
    with pytest.raises(RuntimeError, match="scale must be finite"):
        cuda_attn.paged_attn(q, kc, kc, i, i[0, :1], i[0], scale=float("inf"))
    with pytest.raises(RuntimeError, match="dtype"):
        cuda_attn.paged_read(kc, kc, i, i[0, :1], i[0], 1, dtype=torch.float32)


def test_page_pool():
    from cuda_attn.serve_paged import PagePool
    pool = PagePool(6, 16)
    assert pool.reserve(1, 33) and len(pool.of[1]) == 3
    assert pool.reserve(1, 40) and len(pool.of[1]) == 3        # nothing more to give
    assert pool.reserve(2, 16) and len(pool.of[2]) == 1
    assert not pool.reserve(3, 48) and len(pool.free) == 2     # not enough: nothing taken
    assert len({p for s in pool.of.values() for p in s}) == 4  # no page twice
    pool.release(1)
    assert pool.reserve(3, 80) and not pool.free
    pool.release(2), pool.release(3)
    assert sorted(pool.free) == list(range(6))


@pytest.mark.parametrize("scale", [1e-50, -1e-46, 0.0, 1e39, -1e300, float("nan"), float("-inf")])
def test_scales_that_float32_does_not_hold(scale):
    """The library takes a float, and 0 for the default."""
    kc = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    i = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="scale must be finite and not zero"):
        cuda_attn.paged_attn(torch.zeros(1, 4, 64, dtype=torch.float16), kc, kc, i, i[0, :1], i[0], scale=scale)


def test_scales_that_the_kernels_cannot_use(lib):
    """They multiply it with log2(e) first. (Before anything else is looked at; scales in range pass, to the next refusal.)"""
    for scale, text in ((3e38, "scale must be finite"), (-3e38, "scale must be finite"), (float("inf"), "scale must be finite"),
                        (float("nan"), "scale must be finite"), (2e38, "null cache"), (1e-40, "null cache")):
        rc = lib.lib.phantom_attn_paged(None, 4096, 512, 64, 4096, 3, 8, F16, 1, scale, 0, None)
        assert rc == ERR_INVALID and text in lib.last_error(), (scale, lib.last_error())


def test_requests_that_could_never_run_are_refused():
    """They would wait at the head of the queue for good, and all behind them."""
    from cuda_attn.serve_paged import Server
    with pytest.raises(ValueError, match="at least one token"):
        Server(heads=1, group=1, d=64, chunk=0, device="cpu")
    s = Server(heads=1, group=1, d=64, page=16, pages=5, vocab=50, device="cpu")
    for prompt, want, text in (([1] * 70, 11, "exceed the pool"), ([1] * 81, 1, "exceed the pool"), ([], 3, "needs a prompt"),
                               ([1, 2], 0, "at least one token"), ([1, 50], 2, "from 0 to 49"), ([-1], 2, "from 0 to 49")):
        with pytest.raises(ValueError, match=text):
            s.submit(prompt, want)
    assert not s.waiting and not s.requests and s.step() == []
    s.submit([1] * 70, 10)
    assert s.pool.reserve(99, 16)  # a finished sequence that nobody released
    with pytest.raises(RuntimeError, match="released"):
        s.step()


def test_serving_command_refuses_a_pool_that_is_too_small(monkeypatch, capsys):
    from cuda_attn import serve_paged

    def small(requests, **kw):
        serve_paged.Server(heads=1, group=1, d=64, device="cpu", page=kw["page"], pages=kw["pages"]).submit([1] * 900, 39)
    monkeypatch.setattr(serve_paged, "run", small)
    with pytest.raises(SystemExit) as e:
        serve_paged.main(["--pages", "50"])
    assert e.value.code == 2 and "exceed the pool of 50 pages" in capsys.readouterr().err
