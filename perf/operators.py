"""Cases and plain forms of the state-space operators: the short causal convolution, the selective scan
(prompts and single tokens) and the gated group norm.

``run`` computes them in elementary torch operations where ``own`` is false, and through the package's
entry points where it is true.
"""
import math
import random
import sys

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CHUNK = 64  # chunk length of the plain scan


# ---------------------------------------------------------------- cases
def listed():
    return [
        # the convolution in front of the gated delta rule at the text-prefill shape: 2 x 16 x 128 + 32 x 128 channels
        dict(name="conv_text", op="conv", dtype="bf16", n=1, t=1141, packed=False, c=8192, w=4, bias=False, silu=True, s0=True),
        # a packed batch of prompts, lengths 200 to 4096, of a layer with 64 heads of 64 and 8 groups of 128
        dict(name="conv_packed", op="conv", dtype="bf16", n=8, t=4096, packed=True, mix=1, c=6144, w=4, bias=True, silu=True, s0=True),
        # odd sizes in fp32: channels that no wide load divides, three taps, no activation
        dict(name="conv_odd_fp32", op="conv", dtype="fp32", n=3, t=517, packed=False, c=1027, w=3, bias=True, silu=False, s0=False),
        # single tokens of 64 requests
        dict(name="conv_decode", op="conv_decode", dtype="bf16", n=64, t=1, c=8192, w=4, bias=True, silu=True),
        # the scan at the text-prefill shape: 32 heads of 128, state 128, 16 groups
        dict(name="scan_text", op="scan", n=1, t=1141, packed=False, h=32, p=128, g=16, s=128, dt="fp32", s0=True, d=True),
        # a packed batch of 8 prompts, 64 heads of 64, 8 groups
        dict(name="scan_packed", op="scan", n=8, t=4096, packed=True, mix=2, h=64, p=64, g=8, s=128, dt="bf16", s0=True, d=True),
        # one long stream on a shard of 4 heads
        dict(name="scan_long", op="scan", n=1, t=65536, packed=False, h=4, p=128, g=2, s=128, dt="fp32", s0=False, d=True),
        # throughput: a batch of prompts, all heads on one group
        dict(name="scan_batch", op="scan", n=8, t=4096, packed=False, h=64, p=64, g=1, s=128, dt="bf16", s0=True, d=True),
        # one request's next token: latency
        dict(name="scan_decode_one", op="scan_decode", n=1, t=1, h=32, p=128, g=16, s=128, dt="fp32", d=True),
        # the next token of 128 requests: the states' bytes
        dict(name="scan_decode_batch", op="scan_decode", n=128, t=1, h=64, p=64, g=8, s=128, dt="bf16", d=True),
        # the norm of one request's next tokens
        dict(name="norm_decode", op="norm", dtype="fp16", rows=16, c=4096, g=8),
        # the norm of a batch of prompts
        dict(name="norm_prompt", op="norm", dtype="bf16", rows=32768, c=4096, g=1),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["conv", "conv_decode", "scan", "scan", "scan", "scan_decode", "norm"])
    if op == "conv":
        c = _log(rng, 16, 8192)
        n = _log(rng, 1, 16)
        return dict(op=op, dtype=rng.choice(["bf16", "fp16", "fp32"]), n=n, t=_log(rng, 1, max(1, min(4096, 80_000_000 // (n * c)))),
                    packed=rng.random() < 0.5, mix=rng.randrange(1000), c=c, w=rng.choice([2, 3, 4]), bias=rng.random() < 0.5, silu=rng.random() < 0.7,
                    s0=rng.random() < 0.5)
    if op == "conv_decode":
        return dict(op=op, dtype=rng.choice(["bf16", "fp16", "fp32"]), n=_log(rng, 1, 256), t=rng.choice([1, 1, 1, 3]),
                    c=_log(rng, 16, 8192), w=rng.choice([2, 3, 4]), bias=rng.random() < 0.5, silu=rng.random() < 0.7)
    if op == "norm":
        g = rng.choice([1, 2, 4, 8])
        c = g * _log(rng, 8, 8192 // g)
        return dict(op=op, dtype=rng.choice(["bf16", "fp16", "fp32"]), rows=_log(rng, 1, min(65536, 60_000_000 // c)), c=c, g=g)
    g = rng.choice([1, 1, 2, 4, 8])
    h = g * _log(rng, 1, 64 // g)
    p = rng.choice([32, 64, 64, 64, 80, 96, 128, 128])
    s = rng.choice([16, 64, 64, 96, 128, 128, 128])
    if op == "scan_decode":
        return dict(op=op, n=_log(rng, 1, max(1, 8192 // h)), t=rng.choice([1, 1, 1, 2]), h=h, p=p, g=g, s=s,
                    dt=rng.choice(["fp32", "bf16"]), d=rng.random() < 0.7)
    n = _log(rng, 1, 16)
    t = _log(rng, 1, max(1, min(65536, 60_000_000 // (n * h * p))))
    return dict(op=op, n=n, t=t, packed=rng.random() < 0.5, mix=rng.randrange(1000), h=h, p=p, g=g, s=s, dt=rng.choice(["fp32", "bf16"]),
                s0=rng.random() < 0.5, d=rng.random() < 0.7)


def _lengths(case):
    """Lengths of the sequences; a packed batch's are uniform from a twentieth of t to t, one of them t."""
    if not case.get("packed"):
        return [case["t"]] * case["n"]
    r = random.Random(case["mix"])
    lens = [r.randint(case["t"] // 20, case["t"]) for _ in range(case["n"])]
    lens[r.randrange(case["n"])] = case["t"]
    return lens


def work(case):
    if case["op"] == "norm":
        b = 4 if case["dtype"] == "fp32" else 2
        e = case["rows"] * case["c"]
        return {"bytes": 3 * e * b + case["c"] * b, "flops": 10 * e}
    tokens = sum(_lengths(case))
    if case["op"] in ("conv", "conv_decode"):
        b = 4 if case["dtype"] == "fp32" else 2
        state = case["n"] * (case["w"] - 1) * case["c"] * b
        e = tokens * case["c"]
        reads = state if case["op"] == "conv_decode" or case["s0"] else 0
        return {"bytes": 2 * e * b + reads + state + case["c"] * case["w"] * b, "flops": 2 * case["w"] * e}
    state = case["n"] * case["h"] * case["p"] * case["s"] * 4
    reads = state if case["op"] == "scan_decode" or case["s0"] else 0
    per_token = 4 * case["h"] * case["p"] + 4 * case["g"] * case["s"] + case["h"] * (4 if case["dt"] == "fp32" else 2)
    return {"bytes": tokens * per_token + reads + state, "flops": 4 * tokens * case["h"] * case["p"] * case["s"]}


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(int(seed))

    def nrm(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    def uni(*shape):
        return torch.rand(*shape, generator=gen, device=dev)

    s = dict(case)
    if case["op"] == "norm":
        dtype = DT[case["dtype"]]
        s["x"], s["z"] = nrm(case["rows"], case["c"]).to(dtype), nrm(case["rows"], case["c"]).to(dtype)
        s["wt"] = (1 + 0.1 * nrm(case["c"])).to(dtype)
        return s
    lens = _lengths(case)
    lead = (1, sum(lens)) if case.get("packed") else (case["n"], case["t"])
    s["lens"] = lens
    if case.get("packed"):
        s["cu"] = torch.tensor([0] + lens, device=dev).cumsum(0).to(torch.int32)
    if case["op"] in ("conv", "conv_decode"):
        dtype, c, w = DT[case["dtype"]], case["c"], case["w"]
        s["x"] = nrm(*lead, c).to(dtype)
        s["wt"] = (nrm(c, w) / math.sqrt(w)).to(dtype)
        s["b"] = (0.1 * nrm(c)).to(dtype) if case["bias"] else None
        s["state"] = nrm(case["n"], w - 1, c).to(dtype) if case.get("s0", True) else None
        return s
    h, p, g, n = case["h"], case["p"], case["g"], case["s"]
    s["x"] = nrm(*lead, h, p).bfloat16()
    s["B"], s["C"] = nrm(*lead, g, n).bfloat16(), nrm(*lead, g, n).bfloat16()
    s["dtv"] = (0.5 * nrm(*lead, h)).to(DT[case["dt"]])
    # step sizes whose softplus is spread over 0.001 to 0.1 (log-uniform), decay rates from 1 to 16
    step = torch.exp(uni(h) * math.log(100.0) + math.log(0.001))
    s["dt_bias"] = step + torch.log(-torch.expm1(-step))
    s["A"] = -(1 + 15 * uni(h))
    s["D"] = nrm(h) if case["d"] else None
    s["state"] = 0.5 * nrm(case["n"], h, p, n) if case.get("s0", True) else None
    return s


# ---------------------------------------------------------------- plain forms (32 bits)
def _unpack(x, lens):
    """[1, sum(lens), ...] -> [len(lens), max(lens), ...] with zeros behind each sequence, and the index that goes back."""
    top = max(lens)
    ln = torch.tensor(lens, device=x.device)
    start = ln.cumsum(0) - ln
    pos = torch.arange(top, device=x.device)
    inside = pos[None, :] < ln[:, None]
    src = torch.where(inside, start[:, None] + pos[None, :], 0)
    out = x[0][src] * inside.reshape(inside.shape + (1,) * (x.dim() - 2)).to(x.dtype)
    return out, inside


def _silu(v):
    return v / (1 + torch.exp(-v))


def _softplus(v):
    return torch.where(v > 20, v, torch.log1p(torch.exp(v)))


def _conv_plain(s):
    x = s["x"].float()
    inside = None
    if s.get("packed"):
        x, inside = _unpack(x, s["lens"])
    n, t, c = x.shape
    w = s["w"]
    before = s["state"].float() if s["state"] is not None else x.new_zeros(n, w - 1, c)
    xp = torch.cat([before, x], 1)
    wt = s["wt"].float()
    y = sum(xp[:, j:j + t] * wt[:, j] for j in range(w))
    if s["b"] is not None:
        y = y + s["b"].float()
    if s["silu"]:
        y = _silu(y)
    ln = torch.tensor(s["lens"], device=x.device)
    last = ln[:, None] + torch.arange(w - 1, device=x.device)[None, :]
    tail = xp[torch.arange(n, device=x.device)[:, None], last].to(s["x"].dtype)
    y = y.to(s["x"].dtype)
    return (y[inside][None] if inside is not None else y), tail


def _scan_plain(s):
    x, B, C, dtv = s["x"].float(), s["B"].float(), s["C"].float(), s["dtv"].float()
    inside = None
    d = _softplus(dtv + s["dt_bias"])
    if s.get("packed"):
        (x, inside), (B, _), (C, _), (d, _) = (_unpack(v, s["lens"]) for v in (x, B, C, d))
    n, t, h, p = x.shape
    g, ns = B.shape[2], B.shape[3]
    nc, r = -(-t // CHUNK), h // g

    def chunks(v):  # [n, t, a, b] -> [n, a, nc, CHUNK, b]
        v = torch.cat([v, v.new_zeros(n, nc * CHUNK - t, *v.shape[2:])], 1)
        return v.reshape(n, nc, CHUNK, *v.shape[2:]).transpose(2, 3).transpose(1, 2)

    xc, Bc, Cc, dc = chunks(x), chunks(B), chunks(C), chunks(d[..., None])[..., 0]
    c = (dc.double() * s["A"].double()[None, :, None, None]).cumsum(-1)  # [n, h, nc, CHUNK]
    tri = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=x.device).tril()
    L = torch.exp((c[..., :, None] - c[..., None, :]).masked_fill(~tri, -math.inf).float())
    xd = xc * dc[..., None]
    heads = lambda v: v[:, :, None].expand(n, g, r, *v.shape[2:]).reshape(n, h, *v.shape[2:])  # noqa: E731
    M = heads(Cc @ Bc.transpose(-1, -2)) * L
    y = M @ xd
    xe = xd * torch.exp((c[..., -1:] - c).float())[..., None]
    local = xe.transpose(-1, -2) @ heads(Bc)  # [n, h, nc, p, ns]
    # entry state of each chunk: the sum over the earlier chunks' states, decayed, and the initial state
    end = c[..., -1].cumsum(-1)
    begin = torch.cat([torch.zeros_like(end[..., :1]), end[..., :-1]], -1)
    low = torch.ones(nc + 1, nc, dtype=torch.bool, device=x.device).tril(-1)
    at = torch.cat([begin, end[..., -1:]], -1)  # before each chunk, and behind the last
    W = torch.exp((at[..., :, None] - end[..., None, :]).masked_fill(~low, -math.inf).float())
    E = (W @ local.reshape(n, h, nc, p * ns)).reshape(n, h, nc + 1, p, ns)
    if s["state"] is not None:
        E = E + torch.exp(at.float())[..., None, None] * s["state"].float()[:, :, None]
    y = y + torch.exp(c.float())[..., None] * (heads(Cc) @ E[:, :, :-1].transpose(-1, -2))
    y = y.transpose(1, 2).transpose(2, 3).reshape(n, nc * CHUNK, h, p)[:, :t]
    if s["D"] is not None:
        y = y + s["D"][:, None] * x
    y = y.bfloat16()
    return (y[inside][None] if inside is not None else y), E[:, :, -1].contiguous()


def _norm_plain(s):
    x, z, wt = s["x"].float(), s["z"].float(), s["wt"].float()
    u = (x * _silu(z)).reshape(s["rows"], s["g"], -1)
    u = u * torch.rsqrt((u * u).mean(-1, keepdim=True) + 1e-6)
    return (wt * u.reshape(s["rows"], s["c"])).to(s["x"].dtype)


def _package():
    if "qwen-drive-edge-orin_b200" not in sys.path:
        sys.path.insert(0, "qwen-drive-edge-orin_b200")
    import gdn_b200
    return gdn_b200


def run(s):
    if own:
        m = _package()
        if s["op"] == "norm":
            return m.gated_group_rmsnorm(s["x"], s["z"], s["wt"], groups=s["g"], eps=1e-6)
        if s["op"] == "conv":
            if s["packed"]:
                return m.causal_conv_prefill_varlen(s["x"], s["wt"], s["cu"], bias=s["b"], s0=s["state"], silu=s["silu"])
            return m.causal_conv_prefill(s["x"], s["wt"], bias=s["b"], s0=s["state"], silu=s["silu"])
        if s["op"] == "conv_decode":
            return [m.causal_conv_decode(s["x"], s["wt"], s["state"], bias=s["b"], silu=s["silu"]), s["state"]]
        kw = dict(D=s["D"], dt_bias=s["dt_bias"], dt_softplus=True)
        if s["op"] == "scan_decode":
            return [m.selective_scan_decode(s["x"], s["dtv"], s["A"], s["B"], s["C"], s["state"], **kw), s["state"]]
        if s["packed"]:
            return m.selective_scan_prefill_varlen(s["x"], s["dtv"], s["A"], s["B"], s["C"], s["cu"], s0=s["state"], **kw)
        return m.selective_scan_prefill(s["x"], s["dtv"], s["A"], s["B"], s["C"], s0=s["state"], **kw)
    if s["op"] == "norm":
        return _norm_plain(s)
    y, state = _conv_plain(s) if s["op"] in ("conv", "conv_decode") else _scan_plain(s)
    if s["op"] in ("conv_decode", "scan_decode"):  # the state is updated in place
        s["state"].copy_(state)
        return [y, s["state"]]
    return [y, state]


# ---------------------------------------------------------------- 64 bits, from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x, z = s["x"].double(), s["z"].double()
        u = (x * z * torch.sigmoid(z)).unflatten(1, (s["g"], -1))
        u = u / torch.sqrt(u.square().mean(2, keepdim=True) + 1e-6)
        return u.flatten(1) * s["wt"].double()
    pieces = s["x"].split(s["lens"], 1) if case.get("packed") else s["x"].split(1, 0)
    if case["op"] in ("conv", "conv_decode"):
        ys, tails = [], []
        for i, xi in enumerate(pieces):  # each sequence by itself
            past = s["state"][i:i + 1] if s["state"] is not None else xi.new_zeros(1, s["w"] - 1, s["c"])
            row = torch.cat([past, xi], 1)
            tails.append(row[:, row.shape[1] - (s["w"] - 1):].double())
            if not xi.shape[1]:
                continue
            win = row.double().unfold(1, s["w"], 1)
            v = (win * s["wt"].double()).sum(-1)
            if s["b"] is not None:
                v = v + s["b"].double()
            ys.append(v * torch.sigmoid(v) if s["silu"] else v)
        return [torch.cat(ys, 1 if case.get("packed") else 0), torch.cat(tails, 0)]
    h, p, g, ns = s["h"], s["p"], s["g"], s["s"]
    lens = torch.tensor(s["lens"], device="cuda")
    d = torch.nn.functional.softplus(s["dtv"].double() + s["dt_bias"].double(), threshold=60)
    state = s["state"].double().clone() if s["state"] is not None else torch.zeros(s["n"], h, p, ns, dtype=torch.float64, device="cuda")
    first = torch.cumsum(lens, 0) - lens if case.get("packed") else torch.arange(s["n"], device="cuda") * s["t"]
    rows = lambda v: v.reshape(-1, *v.shape[2:])  # noqa: E731
    x, B, C, d = (rows(s["x"]), rows(s["B"]), rows(s["C"]), rows(d))
    y = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    A = s["A"].double()
    for t in range(max(s["lens"])):  # token by token, all sequences that still have one
        live = [i for i, n in enumerate(s["lens"]) if n > t]
        if len(live) == len(s["lens"]):
            at, st = first + t, state
        else:
            ix = torch.tensor(live, device="cuda")
            at, st = first[ix] + t, state[ix]
        dt_ = d[at]
        inc = (dt_[..., None] * x[at].double())[..., None] * B[at].double().repeat_interleave(h // g, 1)[:, :, None, :]
        st.mul_(torch.exp(dt_ * A)[..., None, None]).add_(inc)
        y[at] = (st @ C[at].double().repeat_interleave(h // g, 1)[..., None])[..., 0]
        if st is not state:
            state[ix] = st
    if s["D"] is not None:
        y += s["D"].double()[:, None] * x.double()
    return [y.reshape(s["x"].shape), state]
