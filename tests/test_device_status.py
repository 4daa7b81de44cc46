"""Device timeouts reach the caller.

Every wait in the library's kernels is bounded; one that runs out records
PF_ERR_TIMEOUT in the workspace status word and the kernel ends early.
Here a wait is made to run out on purpose the only safe way: the library's
own wait loop on a barrier that no thread completes, with a 50 ms limit
(pf_wait_selftest).  No fault, trap or hang is involved; the context stays
usable, which the tests check by running a linear afterwards.
"""
import ctypes

import numpy as np
import pytest
import torch

import oracle
from test_gpu_parity import _g128_qweight, _w, _x, assert_rel

pytestmark = pytest.mark.gpu

META = {"hadamard_rotation": True, "hadamard_block_size": 128}


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import polarflash_b200  # noqa: F401
    torch.cuda.init()


def test_timed_out_wait_is_reported_and_reset():
    from polarflash_b200 import _lib, qlinear
    from polarflash_b200.qweight import workspace_status

    dev = torch.device("cuda")
    ws = torch.zeros(1 << 20, dtype=torch.uint8, device=dev)
    assert workspace_status(ws, counters=True) == (_lib.OK, 0)
    s = torch.cuda.current_stream(dev)
    _lib.check(_lib.load().pf_wait_selftest(ctypes.c_void_p(ws.data_ptr()), 50_000_000,
                                            ctypes.c_void_p(s.cuda_stream)), "pf_wait_selftest")
    st, busy = workspace_status(ws, counters=True)
    assert st == _lib.ERR_TIMEOUT and busy == 0
    assert workspace_status(ws, reset=True)[0] == _lib.ERR_TIMEOUT
    assert workspace_status(ws)[0] == _lib.OK
    # the context is still usable: a linear on the same workspace is correct
    qw, pay, _ = _g128_qweight(_w(512, 2048, 3), 3)
    x = _x(1, 2048, 4)
    y = qlinear(qw, x.cuda(), workspace=ws).cpu().numpy()
    assert_rel(y, oracle.linear("int3_g128", pay, 512, 2048, META, x.float().numpy()))
    assert workspace_status(ws, counters=True) == (_lib.OK, 0)


def test_engine_check_raises_runtime_error():
    """check_device_status (called by PFlashCUDAEngine.forward_layer after its
    per-layer synchronisation) turns a recorded timeout into RuntimeError, as
    the reference reports driver failures, and re-arms the workspace."""
    from polarflash_b200 import _lib, qlinear
    from polarflash_b200.qweight import check_device_status, workspace

    dev = torch.device("cuda")
    s = torch.cuda.Stream(device=dev)
    ws = workspace(dev, 1 << 20, s)
    _lib.check(_lib.load().pf_wait_selftest(ctypes.c_void_p(ws.data_ptr()), 20_000_000,
                                            ctypes.c_void_p(s.cuda_stream)), "pf_wait_selftest")
    with pytest.raises(RuntimeError, match="timed out"):
        check_device_status(dev, s)
    check_device_status(dev, s)  # reset: nothing left to report
    qw, pay, _ = _g128_qweight(_w(256, 1024, 9), 2)
    x = _x(2, 1024, 5)
    with torch.cuda.stream(s):
        y = qlinear(qw, x.cuda())
    s.synchronize()
    assert_rel(y.cpu().numpy(), oracle.linear("int2_g128", pay, 256, 1024, META, x.float().numpy()))
    check_device_status(dev, s)
    assert np.isfinite(y.cpu().numpy()).all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("wait_ns", [0, 2000, 20000])
def test_prompt_attention_that_gives_up_leaves_nothing_behind(hd, wait_ns):
    """Waits of the prompt kernel that give up at once, or in the middle: the
    status word says so, every row is right or NaN, and the blocks that come
    behind on the same multiprocessors, whose shared memory a copy still in
    flight would have overwritten, and later calls give what they give alone."""
    from polarflash_b200 import _lib, prompt_attention
    from polarflash_b200.serving import check_serving_status

    g = torch.Generator(device="cuda").manual_seed(hd)
    lens = [700, 90, 1, 1500, 300] * 4
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
    q, k, v = (torch.randn(sum(lens), h, hd, generator=g, device="cuda").bfloat16() for h in (8, 2, 2))
    want = prompt_attention(q, k, v, cu)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    T, p = sum(lens), lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731

    def limited(out, limit):
        s = torch.cuda.current_stream()
        return _lib.load().pf_prompt_selftest(p(q), 8 * hd, p(k), 2 * hd, p(v), 2 * hd, p(out), 8 * hd, 2, p(cu), p(cu),
                                              len(lens), T, T, 8, 2, hd, hd ** -0.5, p(status), limit, ctypes.c_void_p(s.cuda_stream))

    out = torch.zeros_like(q)
    assert limited(out, 2_000_000_001) == _lib.ERR_INVALID_ARGUMENT
    for _ in range(3):
        _lib.check(limited(out, wait_ns), "pf_prompt_selftest")
        after = prompt_attention(q, k, v, cu)
        assert torch.equal(after, want)
        gone = out.isnan().all(-1)  # a row of a head is given up as a whole
        assert (gone == out.isnan().any(-1)).all()
        assert torch.equal(out[~gone], want[~gone])
        assert int(status) == (_lib.ERR_TIMEOUT if gone.any() else _lib.OK)
        if wait_ns == 0:
            assert gone.any()
        if gone.any():
            with pytest.raises(RuntimeError, match="timed out"):
                check_serving_status("cuda")
        check_serving_status("cuda")
        status.zero_()
    _lib.check(limited(out, 2_000_000_000), "pf_prompt_selftest")
    assert torch.equal(out, want) and int(status) == _lib.OK


def _captured_first_call(out):
    """In a fresh process: the device's first prompt_attention is captured; each
    replay that gives up is reported once, by whichever stream asks."""
    import polarflash_b200 as P
    from polarflash_b200 import _lib
    from polarflash_b200.serving import check_serving_status

    q = torch.randn(300, 2, 64, device="cuda").half()
    cu = torch.tensor([0, 300], dtype=torch.int32, device="cuda")
    L = _lib.load()
    L.pf_prompt_attention = lambda *a: L.pf_prompt_selftest(*a[:-1], 0, a[-1])
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        P.prompt_attention(q, q, q, cu)
    said = []
    for _ in range(2):
        with torch.cuda.stream(s):
            g.replay()
            for _ in range(2):
                try:
                    check_serving_status("cuda")
                    said.append("ok")
                except RuntimeError as e:
                    said.append(str(e))
    out.put(said)


def test_captured_first_call_that_gives_up_is_reported():
    import torch.multiprocessing as mp

    ctx = mp.get_context("spawn")
    out = ctx.Queue()
    p = ctx.Process(target=_captured_first_call, args=(out,))
    p.start()
    said = out.get(timeout=120)
    p.join(60)
    assert p.exitcode == 0
    assert "timed out" in said[0] and "timed out" in said[2] and said[1] == said[3] == "ok"
