"""A pipeline of the grouped product that stalls, without a GPU fault.

lm_ops_debug_set makes one barrier of lm_mx_matmul's pipeline expect an arrival that never comes, with
a short limit on every wait.  The kernel stops waiting, lets its copies and MMAs end and returns;
lm_ops_sync then reports LM_ERR_DEVICE_TIMEOUT, and the next product is right again.
"""
import time

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from litemind_b200 import _lib, ops  # noqa: E402

LIMIT_NS = 5_000_000

# Every form of the kernel, long enough that every barrier is used more than once around its ring:
# CTA pairs, 16, 32 and 64 rows a tile with three tiles a CTA, and one tile shared by a cluster.
FORMS = {"pair e4m3": ([2048], 4096, 8192, "e4m3"), "pair e2m1": ([2048], 4096, 8192, "e2m1"), "16 rows": ([4] * 64, 1024, 4096, "e4m3"),
         "32 rows": ([16] * 64, 1024, 4096, "e4m3"), "64 rows": ([40] * 64, 1024, 4096, "e4m3"), "64 rows e2m1": ([50] * 64, 1024, 4096, "e2m1"),
         "shared by four": ([1], 200, 40000, "e4m3"), "shared by two": ([128], 9000, 16384, "e4m3")}
STALLS = range(_lib.LM_STALL_FULL, _lib.LM_STALL_TMEM_EMPTY + 1)


def debug(stall, limit_ns):
    lib = _lib.load()
    _lib.check(lib.lm_ops_debug_set(_lib.LM_DEBUG_PRODUCT_STALL, stall))
    _lib.check(lib.lm_ops_debug_set(_lib.LM_DEBUG_WAIT_LIMIT_NS, limit_ns))


@pytest.fixture(params=list(FORMS))
def form(request):
    counts, n, k, fmt = FORMS[request.param]
    g = torch.Generator(device="cuda").manual_seed(n)
    x = ops.mx_quantize(torch.randn(sum(counts), k, generator=g, device="cuda"), fmt)
    w = ops.mx_quantize(torch.randn(len(counts), n, k, generator=g, device="cuda"), "e2m1")
    offsets = torch.tensor([0] + counts, device="cuda").cumsum(0).to(torch.int32)
    want = ops.mx_matmul(x, w, offsets, dtype=torch.float32)
    ops.sync()
    yield request.param, lambda: ops.mx_matmul(x, w, offsets, dtype=torch.float32), want
    debug(0, 0)


@pytest.mark.parametrize("stall", STALLS)
def test_stalled_pipeline_ends_and_is_reported(form, stall):
    name, product, want = form
    if stall == _lib.LM_STALL_TMEM_EMPTY and name.startswith("shared"):
        pytest.skip("a cluster has one tile and never waits for a free accumulator")
    debug(stall, LIMIT_NS)
    t0 = time.perf_counter()
    product()
    with pytest.raises(_lib.LiteMindError) as err:
        ops.sync()
    assert err.value.status == _lib.LM_ERR_DEVICE_TIMEOUT and "lm_ops_sync" in str(err.value)
    assert time.perf_counter() - t0 < 1.5  # a few limits and drains, not the 2 s default
    debug(0, 0)
    ops.sync()  # reported once
    for _ in range(2):
        assert torch.equal(product(), want)
    ops.sync()


@pytest.mark.parametrize("limit_ns", [1, 3000, 20000])
def test_waits_that_run_out_anywhere(form, limit_ns):
    """Limits below what the pipeline needs: it gives up wherever it is, copies and MMAs in flight."""
    _, product, want = form
    debug(0, limit_ns)
    for _ in range(3):
        got = product()
        try:
            ops.sync()
        except _lib.LiteMindError as err:
            assert err.status == _lib.LM_ERR_DEVICE_TIMEOUT
        else:
            assert torch.equal(got, want)
    debug(0, 0)
    assert torch.equal(product(), want)
    ops.sync()


def test_every_stream_is_told():
    """One stream's sync does not take the failure away from another, whichever asks first."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = ops.mx_quantize(torch.randn(4, 256, generator=g, device="cuda"), "e4m3")
    w = ops.mx_quantize(torch.randn(128, 256, generator=g, device="cuda"), "e2m1")
    streams = [torch.cuda.Stream() for _ in range(3)]

    def sync(stream):
        with torch.cuda.stream(stream):
            try:
                ops.sync()
            except _lib.LiteMindError as err:
                assert err.status == _lib.LM_ERR_DEVICE_TIMEOUT
                return True
            return False

    for s in streams:
        sync(s)  # of stalls before this test
    torch.cuda.synchronize()
    for stalled in range(3):
        debug(_lib.LM_STALL_TMEM_FULL, LIMIT_NS)
        with torch.cuda.stream(streams[stalled]):
            ops.mx_matmul(x, w)
        debug(0, 0)
        streams[stalled].synchronize()
        assert [sync(s) for s in streams] == [True] * 3
        assert [sync(s) for s in streams] == [False] * 3
    sync(torch.cuda.current_stream())


def test_replayed_stall_is_told_where_it_ran():
    """A product captured on one stream and replayed on another: the stream that ran it hears of it."""
    x = ops.mx_quantize(torch.randn(4, 256, device="cuda"), "e4m3")
    w = ops.mx_quantize(torch.randn(128, 256, device="cuda"), "e2m1")
    ops.mx_matmul(x, w)
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    debug(_lib.LM_STALL_TMEM_FULL, LIMIT_NS)
    with torch.cuda.graph(graph):
        ops.mx_matmul(x, w)
    debug(0, 0)
    with torch.cuda.stream(other):
        try:
            ops.sync()  # of stalls before this test
        except _lib.LiteMindError:
            pass
        graph.replay()
        with pytest.raises(_lib.LiteMindError) as err:
            ops.sync()
    assert err.value.status == _lib.LM_ERR_DEVICE_TIMEOUT
    with pytest.raises(_lib.LiteMindError):
        ops.sync()
