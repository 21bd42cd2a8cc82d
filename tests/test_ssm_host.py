"""Host-side checks of the state-space operators: the library exports every symbol that
include/gdn_ssm.h declares, and bad arguments are refused before any device work."""
from __future__ import annotations

import ctypes
import re

import pytest
import torch

from conftest import ROOT
import gdn_b200
from gdn_b200 import _lib, binding, ssm
from gdn_b200.ssm import _rows

INVALID = 1  # cudaErrorInvalidValue
P = ctypes.c_void_p(1 << 20)


def test_library_exports_every_declared_symbol():
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "gdn_ssm.h").read_text(), flags=re.S)
    names = set(re.findall(r"\b([a-z_][a-z0-9_]*)\s*\(", text)) - {"defined"}
    assert {"causal_conv_prefill", "selective_scan_prefill", "gated_group_rmsnorm_forward"} <= names
    raw = ctypes.CDLL(str(_lib.library_path()))
    for n in names:
        assert hasattr(raw, n) and n in _lib.SIGNATURES, n


def _conv(**kw):
    a = dict(x=P, xs=64, w=P, bias=None, s0=None, y=P, sf=P, cu=None, N=1, T=4, C=64, W=4, silu=1, dtype=1)
    a.update(kw)
    return gdn_b200.load_library().causal_conv_prefill(*a.values(), None)


@pytest.mark.parametrize("bad", [dict(x=None), dict(w=None), dict(y=None), dict(sf=None), dict(xs=63), dict(N=-1),
                                 dict(T=-1), dict(C=0), dict(W=1), dict(W=5), dict(dtype=3), dict(dtype=-1)])
def test_conv_refuses(bad):
    assert _conv(**bad) == INVALID


def test_empty_calls_are_no_ops():
    lib = gdn_b200.load_library()
    assert _conv(N=0) == 0
    assert lib.causal_conv_decode(P, 64, P, None, P, P, 2, 0, 64, 4, 1, 1, None) == 0
    assert lib.gated_group_rmsnorm_forward(P, 64, P, 64, P, P, 0, 64, 1, 1e-6, 1, None) == 0
    assert _scan(N=0) == 0
    assert _scan_decode(N=0) == 0 and _scan_decode(T=0) == 0


def _scan(**kw):
    a = dict(x=P, xs=128, dt=P, dts=2, dtb=0, A=P, B=P, bs=128, C=P, cs=128, D=None, bias=None, sp=1, s0=None, y=P, sf=P,
             cu=None, N=1, T=4, H=2, P=64, G=1, NS=128, ws=P, wsb=256, scr=P, scrb=1 << 40)
    a.update(kw)
    return gdn_b200.load_library().selective_scan_prefill(*a.values(), None)


@pytest.mark.parametrize("T", [(1 << 31) - 129, 2_120_000_000, 1 << 24])
@pytest.mark.parametrize("n", [1, 2])
def test_scan_scratch_of_the_longest_sequences(T, n):
    """Segments of sequences up to the 2^31 - 129 token rows that a call may have: 64 KB of states (128 rows of 128
    fp32) and two log decays each, at most 64 segments a sequence."""
    T //= n
    size = gdn_b200.load_library().selective_scan_scratch_size(n, T, 0, 1, 8, 1, 8)
    segments = size // 65536
    assert n < segments <= 64 * n and segments % n == 0
    assert size == segments * 65536 + -(-segments * 8 // 256) * 256


def _scan_decode(**kw):
    a = dict(x=P, xs=128, dt=P, dts=2, dtb=0, A=P, B=P, bs=128, C=P, cs=128, D=None, bias=None, sp=1, state=P, y=P,
             N=1, T=4, H=2, P=64, G=1, NS=128)
    a.update(kw)
    return gdn_b200.load_library().selective_scan_decode(*a.values(), None)


COMMON = [dict(x=None), dict(dt=None), dict(A=None), dict(B=None), dict(C=None), dict(y=None), dict(xs=127), dict(xs=132),
          dict(bs=124), dict(cs=130), dict(dts=1), dict(N=-1), dict(T=-1), dict(H=0), dict(G=0), dict(H=3, G=2), dict(P=0),
          dict(P=60), dict(P=136), dict(NS=4), dict(NS=100), dict(NS=136), dict(N=65536), dict(H=65536, P=8, xs=1 << 20),
          dict(x=ctypes.c_void_p((1 << 20) + 8)), dict(B=ctypes.c_void_p((1 << 20) + 2))]


@pytest.mark.parametrize("bad", COMMON + [dict(sf=None), dict(ws=None), dict(wsb=128), dict(s0=ctypes.c_void_p((1 << 20) + 4))])
def test_scan_refuses(bad):
    assert _scan(**bad) == INVALID


@pytest.mark.parametrize("bad", COMMON + [dict(state=None), dict(state=ctypes.c_void_p((1 << 20) + 4))])
def test_scan_decode_refuses(bad):
    assert _scan_decode(**bad) == INVALID


@pytest.mark.parametrize("bad", [dict(x=None), dict(z=None), dict(w=None), dict(y=None), dict(rows=-1), dict(C=0),
                                 dict(groups=0), dict(groups=3), dict(dtype=3), dict(xs=63), dict(zs=63)])
def test_group_norm_refuses(bad):
    a = dict(x=P, xs=64, z=P, zs=64, w=P, y=P, rows=4, C=64, groups=2, eps=1e-6, dtype=1)
    a.update(bad)
    assert gdn_b200.load_library().gated_group_rmsnorm_forward(*a.values(), None) == INVALID


def test_binding_refuses_cpu_tensors():
    bf = torch.bfloat16
    x, w = torch.zeros(1, 4, 8, dtype=bf), torch.zeros(8, 4, dtype=bf)
    with pytest.raises(ValueError):
        gdn_b200.causal_conv_prefill(x, w)
    with pytest.raises(ValueError):
        gdn_b200.causal_conv_decode(x, w, torch.zeros(1, 3, 8, dtype=bf))
    with pytest.raises(ValueError):
        gdn_b200.gated_group_rmsnorm(x, x, torch.zeros(8, dtype=bf))
    xs, b, dt, a = torch.zeros(1, 4, 2, 64, dtype=bf), torch.zeros(1, 4, 1, 64, dtype=bf), torch.zeros(1, 4, 2), torch.zeros(2)
    with pytest.raises(ValueError):
        gdn_b200.selective_scan_prefill(xs, dt, a, b, b)
    with pytest.raises(ValueError):
        gdn_b200.selective_scan_decode(xs, dt, a, b, b, torch.zeros(1, 2, 64, 64))


def test_rows_keeps_slices_and_copies_the_rest():
    wide = torch.arange(2 * 3 * 20.).reshape(2, 3, 20)
    t, s = _rows(wide[..., 4:12], 2)
    assert t.data_ptr() == wide[..., 4:12].data_ptr() and s == 20
    t, s = _rows(wide.transpose(0, 1), 2)  # tokens not evenly spaced
    assert s == 20 and torch.equal(t, wide.transpose(0, 1)) and t.is_contiguous()
    t, s = _rows(wide[..., ::2], 2)  # channels not contiguous
    assert s == 10 and torch.equal(t, wide[..., ::2])
    t, s = _rows(wide[:1, :1].expand(2, 3, 20), 2)  # a broadcast input
    assert s == 20 and t.is_contiguous()
    t, s = _rows(wide[:, 1:2, :8], 2)  # one token per sequence
    assert s == 60 and t.data_ptr() == wide[0, 1].data_ptr()
    t, s = _rows(wide.reshape(-1)[1:113].reshape(14, 8), 1, 4)  # contiguous, misaligned
    assert s == 8 and t.data_ptr() % 16 == 0
    t, s = _rows(torch.zeros(2, 0, 8), 2)
    assert s >= 8


def test_every_call_of_a_scan_runs_on_the_inputs_device(monkeypatch):
    """The scratch is planned for the device that the kernels run on, not for the thread's current one (a fake of
    the library notes which device is current; CPU tensors stand in, whose device index is -1)."""
    current, calls = [0], []

    class On:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            self.before, current[0] = current[0], self.dev

        def __exit__(self, *e):
            current[0] = self.before

    class Lib:
        def selective_scan_scratch_size(self, *a):
            calls.append(("size", current[0]))
            return 512

        def selective_scan_prefill(self, *a):
            calls.append(("launch", current[0]))
            return 0

    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(ssm, "_raw_stream", lambda dev: 0)
    monkeypatch.setattr(ssm, "_on_one_device", lambda *t: -1)
    monkeypatch.setattr(ssm, "_status", lambda dev: 0)
    monkeypatch.setattr(ssm, "load_library", Lib)
    b = torch.zeros(1, 20, 1, 8, dtype=torch.bfloat16)
    gdn_b200.selective_scan_prefill(b, torch.zeros(1, 20, 1), torch.zeros(1), b, b)
    assert calls == [("size", -1), ("launch", -1)] and current == [0]


def test_a_workspace_is_never_replaced(monkeypatch):
    """A captured graph holds the address of the workspace it was captured with: a larger one later leaves it alive,
    the small calls keep using it, and its status word is still read (and cleared) with the larger one's."""
    cache = {}
    monkeypatch.setattr(binding, "_ws_cache", cache)
    monkeypatch.setattr(ssm, "_ws_cache", cache)
    cpu = torch.device("cpu", 0)
    small = binding._workspace(cpu, 256)
    large = binding._workspace(cpu, 4096)
    assert large.numel() >= 4096 and not large.any()
    assert binding._workspace(cpu, 256).data_ptr() == small.data_ptr() == ssm._status(0)
    assert binding._workspace(cpu, 3000).data_ptr() == large.data_ptr()

    class Lib:
        @staticmethod
        def deltanet_read_status(ws, out, clear, stream):
            word = ctypes.cast(ws, ctypes.POINTER(ctypes.c_int))
            out._obj.value = word[0]
            if clear:
                word[0] = 0
            return 0

    class On:
        def __init__(self, dev):
            pass

        def __enter__(self):
            pass

        def __exit__(self, *e):
            pass

    monkeypatch.setattr(binding, "load_library", Lib)
    monkeypatch.setattr(binding, "_stream", lambda: None)
    monkeypatch.setattr(torch.cuda, "device", On)
    small.view(torch.int32)[0], large.view(torch.int32)[0] = 1 | 1 << 16, 1 | 1 << 15
    assert binding.read_status(0, clear=False) == 1 | 1 << 15 | 1 << 16
    assert binding.read_status(0) == 1 | 1 << 15 | 1 << 16
    assert binding.read_status(0) == 0


@pytest.mark.parametrize("bad", [dict(T=15), dict(chunk=-1), dict(ws=None), dict(x=None), dict(scrb=0)])
def test_scan_withheld_load_refuses(bad):
    a = dict(x=P, dt=P, A=P, B=P, C=P, y=P, sf=P, N=1, T=2000, H=2, P=64, G=1, NS=64, ws=P, wsb=256, scr=P, scrb=1 << 40,
             stream=None, chunk=1)
    a.update(bad)
    assert gdn_b200.load_library().selective_scan_test_withheld_load(*a.values()) == INVALID


def test_sizes_that_do_not_fit_the_c_abi_are_refused(monkeypatch):
    """Their low 32 bits would be taken for the size (meta tensors stand in for ones of many GB)."""
    monkeypatch.setattr(ssm, "_on_one_device", lambda *t: -1)
    monkeypatch.setattr(ssm, "load_library", lambda: pytest.fail("called the library"))
    e = lambda *shape, dtype=torch.bfloat16: torch.empty(*shape, dtype=dtype, device="meta")
    big = (1 << 32) + 5
    for shape in ((1, big, 1), (big, 1, 1), (1, 1, big)):
        with pytest.raises(ValueError):
            gdn_b200.causal_conv_prefill(e(*shape), e(shape[2], 4))
        with pytest.raises(ValueError):
            gdn_b200.causal_conv_decode(e(*shape), e(shape[2], 4), e(shape[0], 3, shape[2]))
    for b, T in ((1, big), (1, (1 << 31) - 128), (65535, 1 << 16)):
        args = (e(b, T, 1, 8), e(b, T, 1), e(1, dtype=torch.float32), e(b, T, 1, 8), e(b, T, 1, 8))
        with pytest.raises(ValueError):
            gdn_b200.selective_scan_prefill(*args)
        if T == big:
            with pytest.raises(ValueError):
                gdn_b200.selective_scan_decode(*args, e(b, 1, 8, 8, dtype=torch.float32))
    with pytest.raises(ValueError):
        gdn_b200.gated_group_rmsnorm(e(2, big), e(2, big), e(big))
