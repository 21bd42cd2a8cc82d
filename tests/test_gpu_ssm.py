"""State-space operators on the GPU against plain 64-bit restatements of their formulas.

Tolerances. An output held in a type of half-step e (relative: bf16 2^-8, fp16 2^-11, fp32 2^-24) is
off by at most e |y| from its own rounding; fp32 sums of n terms are off by about n 2^-24 of the sum of
the terms' magnitudes. Each check states its bound from those two.
"""
from __future__ import annotations

import math
import time

import pytest
import torch

import gdn_b200

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def nrm(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def close(got, want, bound):
    """|got - want| <= bound elementwise (bound a tensor or number), NaN nowhere."""
    got = got.double()
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), float((got - want).abs().max()), got.shape)


def silu(v):
    return v * torch.sigmoid(v)


# ---------------------------------------------------------------- causal convolution
def conv_ref(x, w, bias, s0, act):
    """One sequence x [T, C] in 64 bits: (y, terms' magnitude, last W - 1 inputs)."""
    W = w.shape[1]
    past = s0 if s0 is not None else x.new_zeros(W - 1, x.shape[1])
    row = torch.cat([past, x], 0).double()
    T = x.shape[0]
    v = sum(row[j:j + T] * w[:, j].double() for j in range(W))
    mag = sum((row[j:j + T] * w[:, j].double()).abs() for j in range(W))
    if bias is not None:
        v, mag = v + bias.double(), mag + bias.double().abs()
    return (silu(v) if act else v), mag, row[row.shape[0] - (W - 1):]


def conv_bound(y, mag, dtype):
    # W + 1 <= 5 fp32 roundings of terms of size mag, through |silu'| <= 1.1; the exponential and the
    # division add a few fp32 ulp (8 taken); one rounding to the output type
    return HALF[dtype] * y.abs() * 1.01 + 2.0 ** -24 * (6 * 1.1 * mag + 8 * y.abs()) + 1e-30 + (6e-8 if dtype == torch.float16 else 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,C,W,bias,act,s0", [(1, 8, 4, True, True, True), (2, 64, 4, False, True, False), (3, 24, 3, True, False, True),
                                               (65, 1027, 4, True, True, True), (200, 8192, 4, False, True, True), (130, 17, 2, True, True, False)])
def test_conv_prefill(dtype, T, C, W, bias, act, s0):
    g = gen(T * C + W)
    x, w = nrm(g, 3, T, C).to(dtype), nrm(g, C, W).to(dtype)
    b = nrm(g, C).to(dtype) if bias else None
    s = nrm(g, 3, W - 1, C).to(dtype) if s0 else None
    y, sf = gdn_b200.causal_conv_prefill(x, w, bias=b, s0=s, silu=act)
    assert y.dtype == dtype and y.shape == x.shape and sf.shape == (3, W - 1, C)
    for i in range(3):
        ry, mag, tail = conv_ref(x[i], w, b, s[i] if s0 else None, act)
        close(y[i], ry, conv_bound(ry, mag, dtype))
        assert torch.equal(sf[i].double(), tail)


@pytest.mark.parametrize("lens", [[5, 0, 1, 130, 2], [0, 0], [1], [64, 64, 3]])
@pytest.mark.parametrize("C", [96, 33])
def test_conv_packed(lens, C):
    """Empty sequences, lengths below the taps, borders inside a tile, rows behind the last one."""
    g, W, tail = gen(sum(lens) + C), 4, 7
    T = sum(lens) + tail
    x, w, s = nrm(g, 1, T, C).bfloat16(), nrm(g, C, W).bfloat16(), nrm(g, len(lens), W - 1, C).bfloat16()
    x[:, sum(lens):] = float("nan")
    cu = torch.tensor([0] + lens, device=DEV).cumsum(0).int()
    y, sf = gdn_b200.causal_conv_prefill_varlen(x, w, cu, s0=s)
    for i, n in enumerate(lens):
        a = int(cu[i])
        ry, mag, last = conv_ref(x[0, a:a + n], w, None, s[i], True)
        close(y[0, a:a + n], ry, conv_bound(ry, mag, torch.bfloat16))
        assert torch.equal(sf[i].double(), last)


def test_conv_leaves_uncovered_rows_and_reads_slices():
    """Through the C ABI: rows that no sequence covers keep their contents; x is a slice of a wider row."""
    g = gen(5)
    wide = nrm(g, 1, 40, 256).bfloat16()
    x, w = wide[..., 64:192], nrm(g, 128, 4).bfloat16()
    cu = torch.tensor([3, 10, 10, 31], device=DEV, dtype=torch.int32)
    y = torch.full((1, 40, 128), 7.0, device=DEV, dtype=torch.bfloat16)
    sf = torch.empty(3, 3, 128, device=DEV, dtype=torch.bfloat16)
    rc = gdn_b200.load_library().causal_conv_prefill(x.data_ptr(), 256, w.data_ptr(), None, None, y.data_ptr(), sf.data_ptr(),
                                                     cu.data_ptr(), 3, 40, 128, 4, 1, 1, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert (y[0, :3] == 7).all() and (y[0, 31:] == 7).all()
    for i, (a, b) in enumerate([(3, 10), (10, 10), (10, 31)]):
        ry, mag, last = conv_ref(x[0, a:b], w, None, None, True)
        close(y[0, a:b], ry, conv_bound(ry, mag, torch.bfloat16))
        assert torch.equal(sf[i].double(), last)
    y2, _ = gdn_b200.causal_conv_prefill_varlen(x, w, cu)
    assert torch.equal(y2[0, 3:31], y[0, 3:31])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,T,C,W", [(1, 1, 8192, 4), (5, 3, 96, 3), (7, 1, 35, 2)])
def test_conv_decode_continues_a_prefill(dtype, B, T, C, W):
    g = gen(B + T + C)
    x, w, b = nrm(g, B, 9 + T, C).to(dtype), nrm(g, C, W).to(dtype), nrm(g, C).to(dtype)
    whole, last = gdn_b200.causal_conv_prefill(x, w, bias=b)
    _, state = gdn_b200.causal_conv_prefill(x[:, :9], w, bias=b)
    y = gdn_b200.causal_conv_decode(x[:, 9:], w, state, bias=b)
    assert torch.equal(y, whole[:, 9:]) and torch.equal(state, last)


# ---------------------------------------------------------------- selective scan
def scan_inputs(g, lead, H, P, G, N, dt=torch.float32, bias=True, D=True):
    s = dict(x=nrm(g, *lead, H, P).bfloat16(), dt=(0.5 * nrm(g, *lead, H)).to(dt), A=-(0.5 + 15 * torch.rand(H, generator=g, device=DEV)),
             B=nrm(g, *lead, G, N).bfloat16(), C=nrm(g, *lead, G, N).bfloat16())
    s["dt_bias"] = -3 + 2 * nrm(g, H) if bias else None
    s["D"] = nrm(g, H) if D else None
    return s


def scan_ref(x, dt, A, B, C, D=None, dt_bias=None, s0=None, dt_softplus=True):
    """One sequence x [T, H, P] token by token in 64 bits: (y, its terms' magnitude, S, its magnitude)."""
    T, H, P = x.shape
    r = H // B.shape[1]
    d = dt.double() + (dt_bias.double() if dt_bias is not None else 0)
    if dt_softplus:
        d = torch.nn.functional.softplus(d, threshold=60)
    S = s0.double().clone() if s0 is not None else torch.zeros(H, P, B.shape[2], dtype=torch.float64, device=x.device)
    M = S.abs()
    ys, ms = [], []
    for t in range(T):
        b, c = B[t].double().repeat_interleave(r, 0), C[t].double().repeat_interleave(r, 0)
        a = torch.exp(d[t] * A.double())[:, None, None]
        inc = (d[t][:, None] * x[t].double())[..., None] * b[:, None, :]
        S, M = a * S + inc, a * M + inc.abs()
        ys.append((S @ c[..., None])[..., 0])
        ms.append((M @ c.abs()[..., None])[..., 0])
        if D is not None:
            ys[-1] = ys[-1] + D.double()[:, None] * x[t].double()
            ms[-1] = ms[-1] + (D.double()[:, None] * x[t].double()).abs()
    if not T:
        return x.double(), x.double(), S, M
    return torch.stack(ys), torch.stack(ms), S, M


# Bounds of the scan. State: fp32 sums and exponentials, some 2^-19 of the terms' magnitude (decays of
# up to 128 tokens are products or exponentials of fp32 sums: 128 half-steps of 2^-24 at most, and as
# many for the sum's terms). y: the bf16 rounding of y, and bf16 roundings (2^-8 each) of at most one
# operand per product, so 2^-8 of the terms' magnitude.
def check_scan(y, sf, ref):
    ry, my, S, M = ref
    close(sf, S, 2.0 ** -16 * M + 1e-30)
    close(y, ry, 2.0 ** -8 * (ry.abs() + my) * 1.01 + 1e-30)
    if ry.numel() > 200:  # and the roundings are not all one way: a quarter of that bound in the mean square
        off = (y.double() - ry).square().mean().sqrt()
        assert off <= 0.25 * 2.0 ** -8 * (ry.abs() + my).square().mean().sqrt()


@pytest.mark.parametrize("T", [1, 2, 63, 64, 65, 127, 128, 129, 300])
@pytest.mark.parametrize("H,P,G,N", [(4, 64, 1, 128), (2, 128, 2, 128), (3, 64, 1, 64)])
def test_scan_prefill_lengths(T, H, P, G, N):
    g = gen(T + H)
    s = scan_inputs(g, (2, T), H, P, G, N)
    s0 = nrm(g, 2, H, P, N)
    y, sf = gdn_b200.selective_scan_prefill(**s, s0=s0, dt_softplus=True)
    for i in range(2):
        check_scan(y[i], sf[i], scan_ref(s["x"][i], s["dt"][i], s["A"], s["B"][i], s["C"][i], s["D"], s["dt_bias"], s0[i]))


@pytest.mark.parametrize("H,P,G,N", [(1, 8, 1, 8), (2, 16, 1, 24), (6, 40, 2, 80), (5, 80, 1, 96), (4, 96, 4, 16), (2, 120, 1, 128),
                                     (8, 64, 8, 128), (24, 64, 8, 64), (3, 72, 3, 40)])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_scan_prefill_sizes(H, P, G, N, dt):
    g = gen(H * P + N)
    s = scan_inputs(g, (1, 150), H, P, G, N, dt, bias=H % 2 == 0, D=H % 2 == 1)
    y, sf = gdn_b200.selective_scan_prefill(**s, dt_softplus=True)
    check_scan(y[0], sf[0], scan_ref(s["x"][0], s["dt"][0], s["A"], s["B"][0], s["C"][0], s["D"], s["dt_bias"]))


def test_scan_without_softplus_and_with_strong_or_no_decay():
    g = gen(3)
    s = scan_inputs(g, (1, 260), 4, 64, 1, 128, bias=False)
    s["dt"] = s["dt"].abs()
    s["A"] = torch.tensor([0.0, -1e-4, -300.0, -1e30], device=DEV)
    y, sf = gdn_b200.selective_scan_prefill(**s)
    check_scan(y[0], sf[0], scan_ref(s["x"][0], s["dt"][0], s["A"], s["B"][0], s["C"][0], s["D"], dt_softplus=False))


@pytest.mark.parametrize("lens", [[300, 0, 1, 128, 17], [0, 0], [129], [127, 1, 128, 256]])
def test_scan_packed(lens):
    """Empty and one-token sequences, borders inside a tile; NaN rows behind the last sequence and
    infinities in a neighbour stay where they are."""
    g = gen(sum(lens))
    H, P, G, N, tail = 4, 64, 2, 128, 9
    T = sum(lens) + tail
    s = scan_inputs(g, (1, T), H, P, G, N)
    cu = torch.tensor([0] + lens, device=DEV).cumsum(0).int()
    for k in ("x", "B", "C", "dt"):
        s[k][:, sum(lens):] = float("nan")
    s0 = nrm(g, len(lens), H, P, N)
    y, sf = gdn_b200.selective_scan_prefill_varlen(**s, cu_seqlens=cu, s0=s0, dt_softplus=True)
    for i, n in enumerate(lens):
        a = slice(int(cu[i]), int(cu[i]) + n)
        check_scan(y[0, a], sf[i], scan_ref(s["x"][0, a], s["dt"][0, a], s["A"], s["B"][0, a], s["C"][0, a], s["D"], s["dt_bias"], s0[i]))
    if len(lens) > 2:  # a neighbour's NaN and infinities
        b = slice(int(cu[-2]), int(cu[-1]))
        for k, v in (("x", float("nan")), ("B", float("inf")), ("C", float("nan")), ("dt", float("nan"))):
            s[k][:, b] = v
        y2, sf2 = gdn_b200.selective_scan_prefill_varlen(**s, cu_seqlens=cu, s0=s0, dt_softplus=True)
        assert torch.equal(y2[0, :int(cu[-2])], y[0, :int(cu[-2])]) and torch.equal(sf2[:-1], sf[:-1])


def segmented(n, T, packed, H, P, G, N):
    return gdn_b200.load_library().selective_scan_scratch_size(n, T, int(packed), H, P, G, N) > 0


@pytest.mark.parametrize("n,T,H,P,G,N", [(1, 3000, 2, 64, 1, 128), (2, 1500, 3, 72, 1, 40), (1, 1281, 4, 128, 2, 64)])
def test_scan_segments_of_long_sequences(n, T, H, P, G, N):
    """Few long sequences, cut into segments whose states are joined: decays from almost none to strong."""
    assert segmented(n, T, False, H, P, G, N)
    g = gen(T)
    s = scan_inputs(g, (n, T), H, P, G, N)
    s["A"] = -torch.logspace(-3, 1.2, H, device=DEV)
    s0 = nrm(g, n, H, P, N)
    y, sf = gdn_b200.selective_scan_prefill(**s, s0=s0, dt_softplus=True)
    for i in range(n):
        check_scan(y[i], sf[i], scan_ref(s["x"][i], s["dt"][i], s["A"], s["B"][i], s["C"][i], s["D"], s["dt_bias"], s0[i]))


@pytest.mark.parametrize("n,T,H,P,G,N,cut", [(10, 32768, 64, 8, 1, 8, False), (5, 16384, 64, 64, 1, 72, True), (1, 65536, 2, 64, 1, 16, True),
                                             (1, 65536, 4, 72, 2, 128, True)])
@pytest.mark.parametrize("A", [-1e-6, -0.01])
def test_scan_state_of_long_prompts_does_not_drift(n, T, H, P, G, N, cut, A):
    """Inputs of one sign and almost no decay: the state is a sum of tens of thousands of terms, none of which cancel.
    Bound, relative to the state. The tensor cores cut off each partial sum of a chunk's 24 products below its last
    place (2^-23 of it): over a group of g chunks that start from zero, half of 24 g 2^-23, with g <= 4 5.7e-6. The
    chunks' sums join by at most 512 rounded additions, whose errors (2^-24 each, both ways) add up to 4 sqrt(512) 2^-24 =
    5.4e-6 at four standard deviations and more. Decays: logarithms up to some 30, whose fp32 sums are off by a few
    2^-24 of them: 6e-6. In all 2e-5."""
    assert segmented(n, T, False, H, P, G, N) == cut
    g = gen(T + N)
    s = scan_inputs(g, (n, T), H, P, G, N, bias=False, D=False)
    s["x"], s["B"], s["dt"] = s["x"].abs(), s["B"].abs(), 0.01 + 0.1 * s["dt"].abs()
    s["A"] = torch.full((H,), A, device=DEV)
    s0 = nrm(g, n, H, P, N).abs()
    _, sf = gdn_b200.selective_scan_prefill(**s, s0=s0)
    for i in {0, n - 1}:
        c = (s["dt"][i].double() * A).cumsum(0)
        w = torch.exp(c[-1] - c) * s["dt"][i].double()
        for h in (0, H - 1):
            S = (s["x"][i, :, h].double() * w[:, h, None]).T @ s["B"][i, :, h * G // H].double() + torch.exp(c[-1, h]) * s0[i, h].double()
            close(sf[i, h], S, 2e-5 * S)


@pytest.mark.parametrize("T", [130, 3000])
def test_scan_keeps_an_infinite_initial_state(T):
    """Infinities in the initial state stay where they are, with their sign; the rest of the state is as without them."""
    g = gen(T)
    s = scan_inputs(g, (1, T), 2, 64, 1, 128)
    s["A"] = -torch.full((2,), 1e-3, device=DEV)
    s0 = nrm(g, 1, 2, 64, 128)
    _, want = gdn_b200.selective_scan_prefill(**s, s0=s0, dt_softplus=True)
    s0[0, 0, 3, 5], s0[0, 1, 40, 100] = math.inf, -math.inf
    _, sf = gdn_b200.selective_scan_prefill(**s, s0=s0, dt_softplus=True)
    assert sf[0, 0, 3, 5] == math.inf and sf[0, 1, 40, 100] == -math.inf
    ok = torch.isfinite(s0)
    # (the two ways of accumulating differ by the hardware's truncation: 24 steps of 2^-23 a chunk)
    assert ((sf - want).abs()[ok] <= 24 * 24 * 2.0 ** -23 * want[ok].abs().max()).all()


def test_scan_segments_of_a_packed_batch():
    """Segments of sequences of unlike lengths, empty ones among them, NaN behind the last."""
    lens, H, P, G, N = [900, 0, 1, 128, 1700, 257, 0], 2, 64, 1, 64
    g = gen(77)
    T = sum(lens) + 5
    assert segmented(len(lens), T, True, H, P, G, N)
    s = scan_inputs(g, (1, T), H, P, G, N, torch.bfloat16)
    s["A"] = -torch.tensor([0.01, 4.0], device=DEV)
    for k in ("x", "B", "C", "dt"):
        s[k][:, sum(lens):] = float("nan")
    cu = torch.tensor([0] + lens, device=DEV).cumsum(0).int()
    s0 = nrm(g, len(lens), H, P, N)
    y, sf = gdn_b200.selective_scan_prefill_varlen(**s, cu_seqlens=cu, s0=s0, dt_softplus=True)
    for i, n in enumerate(lens):
        a = slice(int(cu[i]), int(cu[i]) + n)
        check_scan(y[0, a], sf[i], scan_ref(s["x"][0, a], s["dt"][0, a], s["A"], s["B"][0, a], s["C"][0, a], s["D"], s["dt_bias"], s0[i]))


@pytest.mark.parametrize("count", [31, 70])
def test_scan_many_packed_sequences(count):
    """More sequences than a warp has lanes, and fewer (which are taken longest first), all short."""
    H, P, G, N = 20, 64, 1, 16
    lens = [(37 * i) % 61 for i in range(count)]
    g = gen(count)
    s = scan_inputs(g, (1, sum(lens)), H, P, G, N)
    cu = torch.tensor([0] + lens, device=DEV).cumsum(0).int()
    y, sf = gdn_b200.selective_scan_prefill_varlen(**s, cu_seqlens=cu, dt_softplus=True)
    for i in range(0, count, 3):
        a = slice(int(cu[i]), int(cu[i + 1]))
        check_scan(y[0, a], sf[i], scan_ref(s["x"][0, a], s["dt"][0, a], s["A"], s["B"][0, a], s["C"][0, a], s["D"], s["dt_bias"]))


def test_scan_offsets_out_of_order_or_range_stay_in_the_buffers():
    """Bad offsets give no defined results but touch nothing outside: the guard rows keep their contents."""
    g = gen(15)
    H, P, G, N, T = 2, 64, 1, 64, 200
    s = scan_inputs(g, (1, T), H, P, G, N)
    for bad in ([0, 500, 100, 200], [-7, 30, 20, 1 << 30], [200, 200, 200, 200]):
        cu = torch.tensor(bad, device=DEV, dtype=torch.int32)
        y, sf = gdn_b200.selective_scan_prefill_varlen(**s, cu_seqlens=cu, dt_softplus=True)
        _, cs = gdn_b200.causal_conv_prefill_varlen(s["x"].flatten(2), nrm(g, H * P, 4).bfloat16(), cu)
        torch.cuda.synchronize()
    assert (sf == 0).all() and (cs == 0).all()  # the last ones: three empty sequences


@pytest.mark.parametrize("bad", [[0, 3000, 0, 3000], [0, 3000, 500, 3000], [0, 3000, -5, 1 << 30, 0, 3000], [3000, 0, 3000, 0, 3000],
                                 [0, 1000, 2000, 3000]])
def test_scan_segments_of_offsets_out_of_order_stay_in_the_scratch(bad):
    """Offsets out of order make overlapping sequences: more segments than the scratch has room for. Through the
    C ABI, with guard words around the scratch, the outputs and the final states."""
    g = gen(16)
    H, P, G, N, T, n, pad = 2, 64, 1, 128, 3000, len(bad) - 1, 1 << 16
    lib = gdn_b200.load_library()
    nbytes = lib.selective_scan_scratch_size(n, T, 1, H, P, G, N)
    assert nbytes > 0
    s = scan_inputs(g, (1, T), H, P, G, N)
    cu = torch.tensor(bad, device=DEV, dtype=torch.int32)
    # enough behind the scratch for every sequence to have T tokens in segments of one chunk
    behind = n * (T // 128 + 1) * H * 64 * 128 * 4
    scratch = torch.full((nbytes + 256 + behind,), 0x5A, device=DEV, dtype=torch.uint8)
    y = torch.full((pad + T * H * P + pad,), 7.0, device=DEV, dtype=torch.bfloat16)
    sf = torch.full((pad + n * H * P * N + pad,), 7.0, device=DEV)
    ws = torch.zeros(256, dtype=torch.uint8, device=DEV)
    rc = lib.selective_scan_prefill(s["x"].data_ptr(), H * P, s["dt"].data_ptr(), H, 0, s["A"].data_ptr(), s["B"].data_ptr(), G * N,
                                    s["C"].data_ptr(), G * N, s["D"].data_ptr(), s["dt_bias"].data_ptr(), 1, None, y[pad:].data_ptr(),
                                    sf[pad:].data_ptr(), cu.data_ptr(), n, T, H, P, G, N, ws.data_ptr(), 256,
                                    scratch[256:].data_ptr(), nbytes, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    assert (scratch[:256] == 0x5A).all() and (scratch[256 + nbytes:] == 0x5A).all()
    for t, size in ((y, T * H * P), (sf, n * H * P * N)):
        assert (t[:pad] == 7).all() and (t[pad + size:] == 7).all()
    assert not ws.any()
    if bad == sorted(bad):  # in order: the room is enough, and the results are right
        for i in range(n):
            a = slice(bad[i], bad[i + 1])
            check_scan(y[pad:pad + T * H * P].view(T, H, P)[a], sf[pad:pad + n * H * P * N].view(n, H, P, N)[i],
                       scan_ref(s["x"][0, a], s["dt"][0, a], s["A"], s["B"][0, a], s["C"][0, a], s["D"], s["dt_bias"]))


def test_scan_step_sizes_at_the_edges():
    """Steps of zero (dt of minus infinity under the softplus), tiny and large ones; a zero initial state."""
    g = gen(19)
    s = scan_inputs(g, (1, 140), 4, 64, 1, 64, bias=False)
    s["dt"][0, 10:40] = float("-inf")
    s["dt"][0, 40:60] = -30.0
    s["dt"][0, 60:70] = 40.0
    y, sf = gdn_b200.selective_scan_prefill(**s, s0=torch.zeros(1, 4, 64, 64, device=DEV), dt_softplus=True)
    ref = scan_ref(s["x"][0], s["dt"][0], s["A"], s["B"][0], s["C"][0], s["D"])
    check_scan(y[0], sf[0], ref)


@pytest.mark.parametrize("step", [1e-10, 1e-13, 1e-25, 1e-30])
@pytest.mark.parametrize("log2", [-60.0, -95.0, -99.5])
def test_scan_tiny_steps_before_a_strong_decay(step, log2):
    """Rows between steps so small and, in the same 32 tokens, a decay just within fp32's range: their outputs
    are small and normal numbers, compared relative to the terms' own size (no D, no initial state)."""
    g = gen(24)
    s = scan_inputs(g, (1, 150), 2, 64, 1, 64, bias=False, D=False)
    s["A"] = torch.tensor([-1.0, -0.5], device=DEV)
    s["dt"] = step * (1 + torch.rand(1, 150, 2, generator=g, device=DEV))
    for t in (20, 60, 149):
        s["dt"][0, t] = log2 * math.log(2.0) / s["A"]
    y, sf = gdn_b200.selective_scan_prefill(**s)
    ry, my, S, M = scan_ref(s["x"][0], s["dt"][0], s["A"], s["B"][0], s["C"][0], dt_softplus=False)
    # the scan's bounds; terms below 2^-126 (the decay's remains) may be lost
    close(sf[0], S, 2.0 ** -16 * M + 1e-36)
    close(y[0], ry, 2.0 ** -8 * (ry.abs() + my) * 1.01 + 1e-36 * 64 * 8)


@pytest.mark.parametrize("size", [300.0, 1e4, 3e6, 1e20])
@pytest.mark.parametrize("kept", [False, True])
def test_scan_after_tokens_that_end_the_past(size, kept):
    """A step so large that nothing before it is left, once with its own input and once with none: the
    tokens behind it in its block see the small steps between them."""
    g = gen(23)
    s = scan_inputs(g, (1, 300), 4, 64, 1, 64, bias=False)
    s["dt"] = 0.02 + 0.1 * s["dt"].abs()
    s["A"] = torch.tensor([-1.0, -0.2, -3.0, -0.01], device=DEV)
    for t in (37, 100, 101, 128, 255):
        s["dt"][0, t] = size / s["A"].abs()
        if not kept:
            s["x"][0, t] = 0
    y, sf = gdn_b200.selective_scan_prefill(**s)
    check_scan(y[0], sf[0], scan_ref(s["x"][0], s["dt"][0], s["A"], s["B"][0], s["C"][0], s["D"], dt_softplus=False))


@pytest.mark.parametrize("name,value,first", [("x", math.nan, 128), ("x", math.inf, 128), ("B", math.nan, 200), ("B", -math.inf, 200),
                                              ("C", math.nan, 200), ("dt", math.nan, 200), ("dt", math.inf, 200)])
def test_scan_values_that_are_not_finite_leave_earlier_tokens(name, value, first):
    g = gen(29)
    s = scan_inputs(g, (1, 300), 2, 64, 1, 64)
    ref = scan_ref(s["x"][0, :first], s["dt"][0, :first], s["A"], s["B"][0, :first], s["C"][0, :first], s["D"], s["dt_bias"])
    _, clean = gdn_b200.selective_scan_prefill(**{k: v[:, :first] if v.dim() > 1 else v for k, v in s.items()}, dt_softplus=True)
    s[name][0, 200] = value
    y, _ = gdn_b200.selective_scan_prefill(**s, dt_softplus=True)
    check_scan(y[0, :first], clean[0], ref)
    assert not torch.isfinite(y[0, 200]).any()


@pytest.mark.parametrize("T", [7, 20, 150, 256, 3000])
def test_scan_decay_rates_of_minus_infinity_and_nan(T):
    """A rate of minus infinity leaves each token its own input, in a partial chunk too; a NaN makes its head NaN
    (outputs and state) and no other's."""
    g = gen(T)
    s = scan_inputs(g, (1, T), 4, 64, 1, 64)
    s["A"] = torch.tensor([-math.inf, -1.0, math.nan, -2.0], device=DEV)
    s0 = nrm(g, 1, 4, 64, 64)
    y, sf = gdn_b200.selective_scan_prefill(**s, s0=s0, dt_softplus=True)
    ry, my, S, M = scan_ref(s["x"][0], s["dt"][0], s["A"], s["B"][0], s["C"][0], s["D"], s["dt_bias"], s0[0])
    for h in (0, 1, 3):
        check_scan(y[0, :, h], sf[0, h], (ry[:, h], my[:, h], S[h], M[h]))
    assert torch.isnan(ry[:, 2]).all() and torch.isnan(S[2]).all()
    assert torch.isnan(y[0, :, 2]).all() and torch.isnan(sf[0, 2]).all()


@pytest.mark.parametrize("T", [14, 15, 16, 17])
def test_scan_short_prompts(T):
    g = gen(T)
    s = scan_inputs(g, (3, T), 4, 64, 2, 128)
    s0 = nrm(g, 3, 4, 64, 128)
    y, sf = gdn_b200.selective_scan_prefill(**s, s0=s0, dt_softplus=True)
    for i in range(3):
        check_scan(y[i], sf[i], scan_ref(s["x"][i], s["dt"][i], s["A"], s["B"][i], s["C"][i], s["D"], s["dt_bias"], s0[i]))


def test_scan_refuses_more_sequences_or_heads_than_a_grid_holds():
    e = lambda *shape: torch.empty(*shape, device=DEV, dtype=torch.bfloat16)
    f = lambda *shape: torch.empty(*shape, device=DEV)
    for b, H in ((65536, 1), (1, 65536)):
        args = (e(b, 1, H, 8), f(b, 1, H), f(H), e(b, 1, 1, 8), e(b, 1, 1, 8))
        with pytest.raises(ValueError):
            gdn_b200.selective_scan_prefill(*args)
        with pytest.raises(ValueError):
            gdn_b200.selective_scan_decode(*args, f(b, H, 8, 8))
    with pytest.raises(ValueError):
        gdn_b200.selective_scan_prefill_varlen(e(1, 1, 1, 8), f(1, 1, 1), f(1), e(1, 1, 1, 8), e(1, 1, 1, 8),
                                               torch.zeros(65537, dtype=torch.int32, device=DEV))


def test_scan_prompt_pieces_equal_one_prompt():
    """A prompt in pieces, each from the last one's state, against the whole: the carried state is exact to fp32."""
    g = gen(23)
    H, P, G, N, T = 6, 64, 2, 128, 700
    s = scan_inputs(g, (1, T), H, P, G, N)
    par = {k: s[k] for k in ("A", "D", "dt_bias")}
    cut = lambda a, b: {k: s[k][:, a:b] for k in ("x", "dt", "B", "C")}  # noqa: E731
    y, sf = gdn_b200.selective_scan_prefill(**s, dt_softplus=True)
    state, ys = None, []
    for a, b in ((0, 3), (3, 130), (130, 131), (131, 600), (600, T)):
        yi, state = gdn_b200.selective_scan_prefill(**cut(a, b), **par, s0=state, dt_softplus=True)
        ys.append(yi)
    ref = scan_ref(s["x"][0], s["dt"][0], s["A"], s["B"][0], s["C"][0], s["D"], s["dt_bias"])
    check_scan(torch.cat(ys, 1)[0], state[0], ref)
    check_scan(y[0], sf[0], ref)


def test_scan_leaves_uncovered_rows():
    """Through the C ABI: rows before the first and behind the last sequence keep their contents."""
    g = gen(8)
    H, P, G, N, T = 2, 64, 1, 64, 300
    s = scan_inputs(g, (1, T), H, P, G, N)
    cu = torch.tensor([5, 140, 290], device=DEV, dtype=torch.int32)
    y = torch.full((1, T, H, P), 7.0, device=DEV, dtype=torch.bfloat16)
    sf = torch.empty(2, H, P, N, device=DEV)
    lib = gdn_b200.load_library()
    ws = torch.zeros(256, dtype=torch.uint8, device=DEV)
    scratch = torch.empty(lib.selective_scan_scratch_size(2, T, 1, H, P, G, N), dtype=torch.uint8, device=DEV)
    rc = lib.selective_scan_prefill(s["x"].data_ptr(), H * P, s["dt"].data_ptr(), H, 0, s["A"].data_ptr(), s["B"].data_ptr(), G * N,
                                    s["C"].data_ptr(), G * N, s["D"].data_ptr(), s["dt_bias"].data_ptr(), 1, None, y.data_ptr(),
                                    sf.data_ptr(), cu.data_ptr(), 2, T, H, P, G, N, ws.data_ptr(), 256, scratch.data_ptr(), scratch.numel(),
                                    torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert (y[0, :5] == 7).all() and (y[0, 290:] == 7).all()
    for i, a in enumerate([slice(5, 140), slice(140, 290)]):
        check_scan(y[0, a], sf[i], scan_ref(s["x"][0, a], s["dt"][0, a], s["A"], s["B"][0, a], s["C"][0, a], s["D"], s["dt_bias"]))


def test_scan_reads_slices_of_one_projection():
    """x, B, C and dt as slices of one row, as the convolution's output and the projection leave them."""
    g = gen(11)
    H, P, G, N, T = 4, 64, 2, 64, 200
    xbc = nrm(g, 2, T, H * P + 2 * G * N + 32).bfloat16()
    x, B, C = xbc[..., :H * P].unflatten(2, (H, P)), xbc[..., H * P:H * P + G * N].unflatten(2, (G, N)), None
    C = xbc[..., H * P + G * N:H * P + 2 * G * N].unflatten(2, (G, N))
    dt = xbc[..., -H:]
    A = -torch.rand(H, generator=g, device=DEV) - 0.5
    y, sf = gdn_b200.selective_scan_prefill(x, dt, A, B, C, dt_softplus=True)
    y2, sf2 = gdn_b200.selective_scan_prefill(x.contiguous(), dt.contiguous(), A, B.contiguous(), C.contiguous(), dt_softplus=True)
    assert torch.equal(y, y2) and torch.equal(sf, sf2)
    y3, sf3 = gdn_b200.selective_scan_prefill(x.transpose(0, 1).contiguous().transpose(0, 1), dt, A, B, C, dt_softplus=True)
    assert torch.equal(y, y3) and torch.equal(sf, sf3)


@pytest.mark.parametrize("H,P,G,N,B,T", [(32, 128, 16, 128, 1, 1), (8, 64, 1, 128, 40, 1), (3, 40, 1, 24, 5, 4), (2, 8, 2, 8, 3, 1)])
def test_scan_decode_continues_a_prefill(H, P, G, N, B, T):
    g = gen(H + B)
    s = scan_inputs(g, (B, 20 + T), H, P, G, N, torch.bfloat16)
    per = {k: v for k, v in s.items() if k in ("x", "dt", "B", "C")}
    par = {k: v for k, v in s.items() if k not in per}
    _, state = gdn_b200.selective_scan_prefill(**{k: v[:, :20] for k, v in per.items()}, **par, dt_softplus=True)
    y = gdn_b200.selective_scan_decode(**{k: v[:, 20:] for k, v in per.items()}, **par, state=state, dt_softplus=True)
    for i in range(min(B, 4)):
        ry, my, S, M = scan_ref(s["x"][i], s["dt"][i], s["A"], s["B"][i], s["C"][i], s["D"], s["dt_bias"])
        check_scan(y[i], state[i], (ry[20:], my[20:], S, M))


# ---------------------------------------------------------------- gated group norm
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,C,groups", [(1, 8, 1), (5, 66, 2), (17, 1024, 8), (3, 4096, 1), (2, 20000, 1), (40, 8192, 2), (3, 1001, 7), (9, 512, 1)])
def test_group_norm(dtype, rows, C, groups):
    g = gen(C)
    x, z, w = nrm(g, rows, C).to(dtype), (2 * nrm(g, rows, C)).to(dtype), nrm(g, C).to(dtype)
    y = gdn_b200.gated_group_rmsnorm(x, z, w, groups=groups, eps=1e-5)
    u = (x.double() * silu(z.double())).unflatten(1, (groups, -1))
    ref = (u / (u.square().mean(-1, keepdim=True) + 1e-5).sqrt()).flatten(1) * w.double()
    # one rounding to the type; the mean's sum (a tree of at most 40 serial adds per thread) and some ten fp32 operations
    close(y, ref, HALF[dtype] * ref.abs() * 1.01 + 64 * 2.0 ** -24 * ref.abs() + (6e-8 if dtype == torch.float16 else 1e-37))


def test_group_norm_slices_shapes_and_zero_rows():
    g = gen(2)
    wide = nrm(g, 2, 7, 300).bfloat16()
    x, z, w = wide[..., :64], wide[..., 100:164], nrm(g, 64).bfloat16()
    y = gdn_b200.gated_group_rmsnorm(x, z, w, groups=2)
    assert y.shape == x.shape
    assert torch.equal(y, gdn_b200.gated_group_rmsnorm(x.contiguous(), z.contiguous(), w, groups=2))
    assert (gdn_b200.gated_group_rmsnorm(torch.zeros_like(x), z, w) == 0).all()
    assert gdn_b200.gated_group_rmsnorm(x[:0], z[:0], w).shape == (0, 7, 64)


# ---------------------------------------------------------------- together
def test_layer_prompt_then_tokens():
    """A layer as it is served: convolution, scan, gated norm over a packed prompt batch, then single
    tokens from the carried states, against the same prompts run with those tokens appended."""
    g = gen(21)
    H, P, G, N, W, lens, more = 4, 64, 2, 64, 4, [70, 1, 200], 3
    width = H * P + 2 * G * N
    w, b, nw = nrm(g, width, W).bfloat16() / 2, nrm(g, width).bfloat16() / 4, 1 + nrm(g, H * P).bfloat16() / 8
    par = dict(A=-(1 + torch.rand(H, generator=g, device=DEV)), D=nrm(g, H), dt_bias=nrm(g, H) - 2, dt_softplus=True)
    full = [(nrm(g, 1, n + more, width).bfloat16(), nrm(g, 1, n + more, H).bfloat16(), nrm(g, 1, n + more, H * P).bfloat16()) for n in lens]

    def split(xbc):
        return (xbc[..., :H * P].unflatten(2, (H, P)), xbc[..., H * P:H * P + G * N].unflatten(2, (G, N)),
                xbc[..., H * P + G * N:].unflatten(2, (G, N)))

    def pack(cut):
        cu = torch.tensor([0] + [v[0][:, cut(n)].shape[1] for v, n in zip(full, lens)], device=DEV).cumsum(0).int()
        return [torch.cat([v[j][:, cut(n)] for v, n in zip(full, lens)], 1) for j in range(3)], cu

    def prompt(ins, cu):
        (xbc, dt, z) = ins
        xbc, cs = gdn_b200.causal_conv_prefill_varlen(xbc, w, cu, bias=b)
        x, B, C = split(xbc)
        y, ss = gdn_b200.selective_scan_prefill_varlen(x, dt, par["A"], B, C, cu, D=par["D"], dt_bias=par["dt_bias"], dt_softplus=True)
        return gdn_b200.gated_group_rmsnorm(y.flatten(2), z, nw, groups=G), cs, ss

    out, cu = pack(lambda n: slice(0, n + more))
    want, wcs, wss = prompt(out, cu)
    ins, cu0 = pack(lambda n: slice(0, n))
    _, cs, ss = prompt(ins, cu0)
    for k in range(more):
        xbc, dt, z = (torch.cat([v[j][:, n + k:n + k + 1] for v, n in zip(full, lens)], 0) for j in range(3))
        x, B, C = split(gdn_b200.causal_conv_decode(xbc, w, cs, bias=b))
        y = gdn_b200.selective_scan_decode(x, dt, par["A"], B, C, ss, D=par["D"], dt_bias=par["dt_bias"], dt_softplus=True)
        got = gdn_b200.gated_group_rmsnorm(y.flatten(2), z, nw, groups=G)
        ref = torch.stack([want[0, int(cu[i]) + n + k] for i, n in enumerate(lens)]).double()
        # each side's scan output is within 2^-8 of its terms (two operands' roundings), the norm passes
        # that on, and rounds once: 4 half-steps of the row's largest value
        close(got[:, 0], ref, 4 * 2.0 ** -8 * ref.abs().amax(-1, keepdim=True))
    assert torch.equal(cs, wcs)
    close(ss, wss.double(), 2.0 ** -14 * wss.abs().amax().double())


def test_conv_feeds_the_gated_delta_rule():
    """The convolution in front of the framework's own prefill and decode, packed and with carried states."""
    g = gen(31)
    HQ, HV, D, lens = 1, 2, 128, [90, 40]
    width = 2 * HQ * D + HV * D
    T = sum(lens)
    w = nrm(g, width, 4).bfloat16() / 2
    mixed = nrm(g, 1, T, width).bfloat16()
    gg, beta = -torch.rand(1, T, HV, generator=g, device=DEV), torch.rand(1, T, HV, generator=g, device=DEV)
    cu = torch.tensor([0] + lens, device=DEV).cumsum(0).int()

    def qkv(m):
        q, k, v = m.split([HQ * D, HQ * D, HV * D], -1)
        unit = lambda t: torch.nn.functional.normalize(t.float().unflatten(2, (HQ, D)), dim=-1).bfloat16()  # noqa: E731
        return unit(q), unit(k), v.unflatten(2, (HV, D))

    y, cs = gdn_b200.causal_conv_prefill_varlen(mixed, w, cu)
    o, sf = gdn_b200.chunk_prefill_varlen(*qkv(y), gg, beta, cu)
    for i, n in enumerate(lens):
        a = slice(int(cu[i]), int(cu[i]) + n)
        yi, ci = gdn_b200.causal_conv_prefill(mixed[:, a], w)
        assert torch.equal(yi, y[:, a]) and torch.equal(ci[0], cs[i])
        oi, si = gdn_b200.chunk_prefill(*qkv(yi), gg[:, a], beta[:, a])
        assert torch.equal(oi, o[:, a]) and torch.equal(si[0], sf[i])
    tok = gdn_b200.causal_conv_decode(nrm(g, 2, 1, width).bfloat16(), w, cs)
    od = gdn_b200.recurrent_decode(*qkv(tok), gg[:, :2].transpose(0, 1).contiguous(), beta[:, :2].transpose(0, 1).contiguous(), sf)
    assert torch.isfinite(od.float()).all()


def test_capture_and_replay():
    """All entry points captured into one graph and replayed on new inputs give the eager results."""
    g = gen(41)
    H, P, G, N = 4, 64, 1, 64
    s = scan_inputs(g, (1, 2000), H, P, G, N)
    assert segmented(1, 2000, False, H, P, G, N)
    d = scan_inputs(g, (2, 1), H, P, G, N)
    cx, w, nx, nw = nrm(g, 1, 300, 64).bfloat16(), nrm(g, 64, 4).bfloat16(), nrm(g, 30, 64).half(), nrm(g, 64).half()
    st, cst = nrm(g, 2, H, P, N), nrm(g, 2, 3, 64).bfloat16()

    def step(state, cstate):
        return [*gdn_b200.selective_scan_prefill(**s, dt_softplus=True), *gdn_b200.causal_conv_prefill(cx, w),
                gdn_b200.selective_scan_decode(**d, state=state, dt_softplus=True),
                gdn_b200.causal_conv_decode(cx[:, :2].transpose(0, 1), w, cstate),
                gdn_b200.gated_group_rmsnorm(nx, nx, nw, groups=4)]

    step(st.clone(), cst.clone())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    a, ca = st.clone(), cst.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = step(a, ca)
    for t in (s["x"], d["x"], cx, nx):
        t.copy_(torch.randn(t.shape, generator=g, device=DEV))
    a.copy_(st), ca.copy_(cst)
    graph.replay()
    b, cb = st.clone(), cst.clone()
    for got, want in zip(outs, step(b, cb)):
        assert torch.equal(got, want)
    assert torch.equal(a, b) and torch.equal(ca, cb)


def test_capture_of_a_first_call(monkeypatch):
    """A capture that makes the device's workspace: its status word is zero at once, and replays keep what other calls
    wrote there."""
    g = gen(43)
    s = scan_inputs(g, (1, 200), 2, 64, 1, 64)
    want = gdn_b200.selective_scan_prefill(**s, dt_softplus=True)  # (loads the kernels)
    torch.full((1 << 20,), 0x5A, dtype=torch.uint8, device=DEV)  # (freed memory that is not zero)
    cache = {}
    monkeypatch.setattr(gdn_b200.binding, "_ws_cache", cache)
    monkeypatch.setattr(gdn_b200.ssm, "_ws_cache", cache)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = gdn_b200.selective_scan_prefill(**s, dt_softplus=True)
    (ws,), = cache.values()
    assert not ws.any()
    ws[0] = 1
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert gdn_b200.binding.read_status() == 1 and gdn_b200.binding.read_status() == 0


def test_streams_run_side_by_side():
    """Calls on two streams at once keep their own results."""
    g = gen(51)
    sets = [scan_inputs(g, (1, 5000), 2, 64, 1, 128) for _ in range(2)]
    want = [gdn_b200.selective_scan_prefill(**s, dt_softplus=True) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(4):
        for i, (st, s) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(st):
                got[i].append(gdn_b200.selective_scan_prefill(**s, dt_softplus=True))
    torch.cuda.synchronize()
    for i in range(2):
        for y, sf in got[i]:
            assert torch.equal(y, want[i][0]) and torch.equal(sf, want[i][1])


@pytest.mark.parametrize("T,cut", [(700, False), (20000, True)])
def test_scan_withheld_load_times_out_and_the_next_call_is_clean(T, cut):
    """Failure detection without a fault: tiles that never arrive. The bounded waits (about 1 s each) run out, the
    status word says so (bit 0, and bit 16 for the scan), the kernels end, and the next call is as before."""
    n, H, P, G, N = (1, 2, 64, 1, 64) if cut else (4, 40, 64, 1, 64)
    lib = gdn_b200.load_library()
    nbytes = lib.selective_scan_scratch_size(n, T, 0, H, P, G, N)
    assert (nbytes > 0) == cut  # (cut: 53 segments of three chunks)
    g = gen(T)
    s = scan_inputs(g, (n, T), H, P, G, N, bias=False, D=False)
    s["dt"] = s["dt"].abs()
    want = gdn_b200.selective_scan_prefill(**s)
    y, sf = torch.empty_like(s["x"]), torch.empty(n, H, P, N, device=DEV)
    ws, scratch = torch.zeros(64, dtype=torch.int32, device=DEV), torch.empty(max(nbytes, 1), dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    start = time.perf_counter()
    rc = lib.selective_scan_test_withheld_load(s["x"].data_ptr(), s["dt"].data_ptr(), s["A"].data_ptr(), s["B"].data_ptr(), s["C"].data_ptr(),
                                               y.data_ptr(), sf.data_ptr(), n, T, H, P, G, N, ws.data_ptr(), 256, scratch.data_ptr(),
                                               nbytes, torch.cuda.current_stream().cuda_stream, 1)
    assert rc == 0
    torch.cuda.synchronize()  # raises if a kernel faulted
    elapsed = time.perf_counter() - start
    print(f"T={T}: status {int(ws[0]):#x} after {elapsed:.2f} s")
    assert int(ws[0]) == 1 | 1 << 16 and not ws[1:].any()
    assert elapsed < 20.0
    got = gdn_b200.selective_scan_prefill(**s)
    assert gdn_b200.binding.read_status() == 0
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
