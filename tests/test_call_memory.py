"""The scratch memory of calls that are several launches.  Two threads may call at the same time (the interpreter lock is
not held inside the library), also on one stream, so no call's scratch may be another's, and it has to live until the call
returns.  Shown here on the CPU with a stand-in for the library; the same on the GPU is in ``test_gpu_threads.py``."""

import threading

import pytest
import torch
from torch.multiprocessing.reductions import StorageWeakRef

import fast_route_b200 as fr
from fast_route_b200 import _lib


class Library:
    """Asks the real library for sizes.  A call of an operator takes part in ``meeting`` (the other thread is then inside
    its own call), and notes its scratch and whether a living tensor still holds that at the end."""

    def __init__(self, real, made):
        self._real, self._made = real, made
        self.meeting = threading.Barrier(2, timeout=60)
        self.scratch = {}

    def __getattr__(self, name):
        return getattr(self._real, name)

    def _call(self, ws, nbytes):
        begin, end = ws, ws + nbytes
        self.meeting.wait()              # both calls are inside the library
        held = any(not ref.expired() and lo <= begin and end <= hi for ref, lo, hi in list(self._made))
        self.scratch[threading.get_ident()] = (begin, end, held)
        self.meeting.wait()
        return 0

    def fr_fp4_gemm(self, *a):
        return self._call(*a[-3:-1])

    def fr_fp4_quantize(self, *a):
        return self._call(*a[-3:-1])


@pytest.fixture
def library(lib, monkeypatch):
    made = []

    def remembering(make):
        def call(*a, **kw):
            t = make(*a, **kw)
            storage = t.untyped_storage()
            made.append((StorageWeakRef(storage), storage.data_ptr(), storage.data_ptr() + storage.nbytes()))
            return t
        return call
    for name in ("empty", "zeros"):
        monkeypatch.setattr(torch, name, remembering(getattr(torch, name)))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(_lib, "require_cuda", lambda *a: None)
    monkeypatch.setattr(_lib, "elsewhere", lambda device: False)
    monkeypatch.setattr(_lib, "stream_ptr", lambda device=None: 0)
    monkeypatch.setattr(_lib, "_workspaces", {})
    fake = Library(lib, made)
    monkeypatch.setattr(_lib, "load", lambda: fake)
    return fake


def _matmul(m):
    a, s = torch.zeros(m, 32, dtype=torch.uint8), torch.zeros(m, 4, dtype=torch.uint8).view(torch.float8_e4m3fn)
    return lambda: fr.matmul_fp4(a, s, a, s)


def _quantize(rows):
    x = torch.zeros(rows, 64)
    return lambda: fr.quantize_fp4(x)


@pytest.mark.parametrize("first,second", [(_matmul(200), _matmul(200)), (_matmul(200), _matmul(9000)),
                                          (_quantize(2000), _quantize(2000)), (_quantize(2000), _matmul(9000)),
                                          (_matmul(130), _quantize(60000))])
def test_two_calls_at_once_have_scratch_of_their_own(library, first, second):
    errors = []

    def go(call):
        try:
            call()
        except BaseException as e:      # noqa: BLE001  (reported below)
            errors.append(e)
            library.meeting.abort()
    threads = [threading.Thread(target=go, args=(c,)) for c in (first, second)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    (a0, a1, a_held), (b0, b1, b_held) = library.scratch.values()
    assert a1 <= b0 or b1 <= a0, "both calls use the same memory"
    assert a_held and b_held, "the memory was given back while its call was running"


def test_a_captured_call_clears_its_state_only(lib, monkeypatch):
    """Inside a capture every replay repeats the clearing: the few-token layer's control words and logits, not the rest."""
    state = lib.fr_moe_decode_state_bytes()
    nbytes = lib.fr_moe_decode_workspace_bytes(16, 2048, 1408, 64, 6)
    assert 0 < state < 40000 < (1 << 20) < nbytes
    for sizes in ((1, 64, 64, 4, 2), (16, 4096, 14336, 256, 8)):        # the state has the same place at every size
        assert lib.fr_moe_decode_workspace_bytes(*sizes) > state
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **kw: empty(*a, **kw).fill_(7))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    ws = _lib.call_workspace(nbytes, torch.device("cpu"), "decode", lib.fr_moe_decode_state_bytes)
    assert ws.numel() == nbytes and ws.data_ptr() % 256 == 0
    assert not ws[:state].any() and (ws[state:] == 7).all()


def test_sizes_that_need_scratch_are_the_librarys(lib):
    """``quantize_fp4`` and ``matmul_fp4`` do not ask the library where it needs no workspace; the limits are its own."""
    from fast_route_b200.ops import fp4
    need = lib.fr_fp4_quantize_workspace_bytes
    assert need(1, 1, fp4._SMALL) == 0 and need(7, fp4._SMALL // 32, 32) == 0
    assert need(1, fp4._SMALL // 32 + 1, 32) > 0 and need(7, fp4._SMALL // 32 + 1, 32) > 0
    for block in (16, 32):
        for n, k in ((1, 32), (5000, 4096)):
            need = lib.fr_fp4_gemm_workspace_bytes
            assert need(1, n, k, block) == need(32, n, k, block) == need(33, n, k, block) == need(128, n, k, block) == 0
            assert need(129, n, k, block) > 0
