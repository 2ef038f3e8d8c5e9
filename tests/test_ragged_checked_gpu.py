"""The ragged kernels in the checked build (build.py --debug): no address or coordinate check
fails over the forms and their edges, and a bounded wait that runs out is reported, ends the
launch and leaves the context and the workspace usable. Called through the C ABI with packed
structs, as an FFI host would."""
import ctypes
import os
import time

import pytest
import torch

from gqa_kernels import _lib
from tests._serving import attention64, check_attention, paged_batch
from tests.test_serving_host import RAGGED

pytestmark = pytest.mark.gpu
GQA_ERR_TIMEOUT = 5
LIMIT_NS = 20_000_000
STREAM_SITES = set(range(111, 115))
TILE_SITES = set(range(121, 148))


@pytest.fixture(scope="module")
def dbg(cuda_lib, lib_path):
    path = os.path.join(os.path.dirname(lib_path), "libgqa_sm100_debug.so")
    assert os.path.exists(path), "build.py --debug first"
    lib = ctypes.CDLL(path)
    for name, (res, args) in _lib.SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args
    return lib


def error(lib):
    code, site = ctypes.c_int(0), ctypes.c_int(0)
    assert lib.gqa_device_error(ctypes.byref(code), ctypes.byref(site), 1) == 0
    return code.value, site.value


def forward(lib, batch, reqs, ws=None, softcap=0.0, window=0, alibi=None, lse=None):
    q, kc, vc, bt, cu, lens = batch
    out = torch.full_like(q, float("nan"))

    def args(ptr, nbytes):
        return RAGGED(ptr, nbytes, q.data_ptr(), kc.data_ptr(), vc.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(),
                      bt.data_ptr(), cu.data_ptr(), lens.data_ptr(), 0 if alibi is None else alibi.data_ptr(), 0, 0,
                      *q.stride(), *kc.stride(), *vc.stride(), *out.stride(), bt.shape[1], lens.shape[0], q.shape[0], q.shape[1],
                      kc.shape[2], q.shape[2], kc.shape[1], kc.shape[0], max(x for x, _ in reqs), max(sum(r) for r in reqs), window, 1,
                      _lib.dtype_code(q), 0, q.shape[2] ** -0.5, softcap, 1.0, 1.0)
    need = lib.gqa_ragged_fwd_workspace_bytes(args(0, 0))
    if ws is None or ws.numel() < need:
        ws = torch.zeros(max(need, 256), dtype=torch.uint8, device="cuda")
    assert lib.gqa_ragged_fwd(args(ws.data_ptr(), ws.numel()), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    return out, ws


@pytest.mark.parametrize("hq,hkv,d,block", [(8, 2, 128, 64), (14, 2, 64, 16), (16, 1, 128, 32)])
@pytest.mark.parametrize("softcap,window", [(0.0, 0), (20.0, 0), (0.0, 150)])
def test_no_check_fails(dbg, hq, hkv, d, block, softcap, window):
    reqs = [(1, 0), (3, 500), (0, 9), (300, 77), (2, 3000), (33, 128), (129, 1)]
    batch = paged_batch(reqs, hq, hkv, d, block, torch.bfloat16, seed=d, poison=float("nan"))
    assert error(dbg) == (0, 0)
    out, _ = forward(dbg, batch, reqs, softcap=softcap, window=window)
    assert error(dbg) == (0, 0)
    q, kc, vc, bt, _, _ = batch
    o, _, a = attention64(q, kc.nan_to_num(0), vc.nan_to_num(0), bt, reqs, softcap=softcap, window=window or None)
    check_attention(out, o, a, torch.bfloat16)


@pytest.mark.parametrize("reqs,load,sites", [
    ([(300, 700)], 2, TILE_SITES),             # pairs of query tiles, K tile 1
    ([(300, 700)], 3, TILE_SITES),             # the same, V tile 1
    ([(20, 100), (20, 3000)], 2, TILE_SITES),  # solo tiles (CTA 0 has the last request)
    ([(40, 16000)], 1, TILE_SITES),            # solo tiles, split keys
    ([(1, 900), (1, 20)], 0, STREAM_SITES), ([(1, 16000)], 1, STREAM_SITES)])
def test_expired_wait_reports_and_recovers(dbg, reqs, load, sites):
    batch = paged_batch(reqs, 8, 2, 128, 64, torch.bfloat16, seed=3)
    ref, _ = forward(dbg, batch, reqs)
    ws = None
    assert error(dbg) == (0, 0)
    assert dbg.gqa_debug_inject(0, load, LIMIT_NS) == 0
    try:
        t0 = time.perf_counter()
        _, ws = forward(dbg, batch, reqs)
        elapsed = time.perf_counter() - t0
        code, site = error(dbg)
    finally:
        assert dbg.gqa_debug_inject(-1, -1, 0) == 0
    assert code == GQA_ERR_TIMEOUT and site in sites, (code, site)
    assert elapsed >= LIMIT_NS * 1e-9
    out, _ = forward(dbg, batch, reqs, ws)
    assert error(dbg) == (0, 0)
    assert torch.equal(out, ref)
