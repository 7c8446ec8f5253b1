"""The 8-bit integer operators of the library as measured cases: int8 weights
from GGUF blocks, RMS norm with the residual's addition into int8, gated
activation into int8, and the int8 matrix product with a scale for each token
and each channel. `run` computes one pass in plain torch operations, or, where
`own` is set, through the library's C entry points."""
import importlib.util
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE_IDS = {"f32": 0, "f16": 1, "bf16": 30}
# GGUF formats: type id, elements and bytes of a block
FORMATS = {"F32": (0, 1, 4), "F16": (1, 1, 2), "Q4_0": (2, 32, 18), "Q4_1": (3, 32, 20), "Q5_0": (6, 32, 22),
           "Q8_0": (8, 32, 34), "Q4_K": (12, 256, 144), "Q5_K": (13, 256, 176), "Q6_K": (14, 256, 210)}
ACTS = {"silu": 0, "gelu": 1, "none": 2}
MAX_MACS = 4096 * 11008 * 4096
MAX_OUT = 1024 * 32000


def listed():
    return [
        # matrix product: one decoded token through q|k|v of a 1.1B model (32 + 2 x 4 heads of 64)
        {"name": "gemm_qkv_1tok", "op": "gemm", "rows": 1, "n": 2560, "k": 2048, "out": "f32", "bias": False},
        # 64 sequences decoded together, gate|up of a 7B model: the weights are what is read
        {"name": "gemm_gateup_64tok", "op": "gemm", "rows": 64, "n": 22016, "k": 4096, "out": "bf16", "bias": False},
        # a prompt of odd length through q|k|v with biases of a 0.5B model
        {"name": "gemm_qkv_bias_333tok", "op": "gemm", "rows": 333, "n": 1152, "k": 896, "out": "f16", "bias": True},
        # long prompts through ffn_down of a 7B model: the largest product
        {"name": "gemm_down_4096tok", "op": "gemm", "rows": 4096, "n": 4096, "k": 11008, "out": "bf16", "bias": False},
        # scoring every position of a text: the logits of 1023 positions
        {"name": "gemm_logits_1023tok", "op": "gemm", "rows": 1023, "n": 32000, "k": 2048, "out": "f32", "bias": False},
        # norm: one decoded token of a 1.1B model, f32 residual stream
        {"name": "norm_1tok", "op": "norm", "rows": 1, "cols": 2048, "type": "f32", "resid": True},
        # a prompt of odd length of a 0.5B model; the first norm has nothing to add
        {"name": "norm_1531tok_896", "op": "norm", "rows": 1531, "cols": 896, "type": "f16", "resid": False},
        # long prompts of a 7B model, the residual added on the way
        {"name": "norm_4096tok_4096", "op": "norm", "rows": 4096, "cols": 4096, "type": "bf16", "resid": True},
        # gated activation: 64 decoded sequences, gate and up of one product side by side
        {"name": "glu_64tok_11008", "op": "glu", "rows": 64, "cols": 11008, "type": "f16", "act": "silu", "up": True},
        # long prompts of a 7B model
        {"name": "glu_4096tok_11008", "op": "glu", "rows": 4096, "cols": 11008, "type": "bf16", "act": "silu", "up": True},
        # int8 weights when a model is loaded: gate of a 1.1B model, ffn_down of a 7B model
        {"name": "weights_q4k_5632x2048", "op": "weights", "format": "Q4_K", "rows": 5632, "cols": 2048},
        {"name": "weights_q8_4096x11008", "op": "weights", "format": "Q8_0", "rows": 4096, "cols": 11008},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)) - 0.5 / lo))))


def draw(rng):
    op = rng.choice(["gemm", "gemm", "gemm", "norm", "glu", "weights"])
    if op == "gemm":
        while True:
            m, n, k = _log_int(rng, 1, 4096), _log_int(rng, 64, 32000), _log_int(rng, 64, 11008)
            if rng.random() < 0.5:
                n, k = max(64, n // 64 * 64), max(64, k // 64 * 64)
            if m * n * k <= MAX_MACS and m * n <= MAX_OUT:
                return {"op": op, "rows": m, "n": n, "k": k, "out": rng.choice(list(DTYPES)), "bias": rng.random() < 0.4}
    if op == "norm":
        while True:
            m, c = _log_int(rng, 1, 32768), _log_int(rng, 64, 8192)
            if rng.random() < 0.5:
                c = max(64, c // 64 * 64)
            if m * c <= 4096 * 4096:
                return {"op": op, "rows": m, "cols": c, "type": rng.choice(list(DTYPES)), "resid": rng.random() < 0.7}
    if op == "glu":
        while True:
            m, c = _log_int(rng, 1, 8192), _log_int(rng, 64, 14336)
            if rng.random() < 0.5:
                c = max(64, c // 64 * 64)
            if m * c <= 4096 * 11008:
                act = rng.choice(list(ACTS))
                return {"op": op, "rows": m, "cols": c, "type": rng.choice(list(DTYPES)), "act": act,
                        "up": rng.random() < 0.6}
    fmt = rng.choice(list(FORMATS))
    step = max(32, FORMATS[fmt][1])
    while True:
        r, c = _log_int(rng, 64, 32000), _log_int(rng, 256, 11008) // step * step
        if r * c <= 4096 * 11008:
            return {"op": op, "format": fmt, "rows": r, "cols": c}


def _pitch(n):
    return (n + 15) // 16 * 16


def _quantised(g, rows, cols):
    """int8 rows of a roughly normal matrix with a scale for each, in a pitch
    of a multiple of 16 whose padding is not zero."""
    q = torch.empty(rows, _pitch(cols), dtype=torch.float16, device="cuda").normal_(generator=g).mul_(30)
    q = q.round_().clamp_(-127, 127).to(torch.int8)
    scale = torch.rand(rows, generator=g, device="cuda").mul_(0.01).add_(0.005)
    return q, scale


def _blocks(g, fmt, rows, cols):
    _, be, bb = FORMATS[fmt]
    if fmt in ("F32", "F16"):
        w = torch.randn(rows, cols, generator=g, device="cuda").mul_(0.02)
        return w.to(torch.float16 if fmt == "F16" else torch.float32).view(torch.uint8).reshape(rows, -1)
    nb = cols // be
    raw = torch.randint(0, 256, (rows, nb, bb), generator=g, device="cuda", dtype=torch.uint8)
    d = torch.rand(rows, nb, 2, generator=g, device="cuda").mul_(3e-3).add_(1e-3).to(torch.float16)
    d = d.view(torch.uint8).reshape(rows, nb, 4)
    if fmt == "Q6_K":
        raw[..., 208:210] = d[..., :2]
        raw[..., 192:208] = torch.randint(-63, 64, (rows, nb, 16), generator=g, device="cuda", dtype=torch.int8).view(torch.uint8)
    elif fmt in ("Q4_K", "Q5_K", "Q4_1"):
        raw[..., :4] = d
    else:
        raw[..., :2] = d[..., :2]
    return raw.reshape(rows, nb * bb)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, s = case["op"], dict(case)
    if op == "gemm":
        m, n, k = case["rows"], case["n"], case["k"]
        s["a"], s["a_scale"] = _quantised(g, m, k)
        s["w"], s["w_scale"] = _quantised(g, n, k)
        s["w_scale"].mul_(0.1)
        s["b"] = torch.randn(n, generator=g, device="cuda").mul_(0.02) if case["bias"] else None
        s["y"] = torch.empty(m, n, dtype=DTYPES[case["out"]], device="cuda")
        return s
    if op == "weights":
        m, c = case["rows"], case["cols"]
        s["raw"] = _blocks(g, case["format"], m, c)
    else:
        m, c, dt = case["rows"], case["cols"], DTYPES[case["type"]]
        if op == "norm":
            s["x"] = torch.randn(m, c, generator=g, device="cuda").to(dt)
            s["r"] = torch.randn(m, c, generator=g, device="cuda").mul_(3).to(dt) if case["resid"] else None
            s["w"] = torch.randn(c, generator=g, device="cuda").mul_(0.05).add_(1)
            s["sum"] = torch.empty(m, c, dtype=dt, device="cuda") if case["resid"] else None
        else:
            # gate and up as one product leaves them: side by side in each row
            s["gu"] = torch.randn(m, c * (2 if case["up"] else 1), generator=g, device="cuda").mul_(1.5).to(dt)
    s["q"] = torch.empty(m, _pitch(c), dtype=torch.int8, device="cuda")
    s["scale"] = torch.empty(m, dtype=torch.float32, device="cuda")
    s["values"] = torch.empty(m, c, dtype=torch.bfloat16, device="cuda")
    return s


# ---------------------------------------------------------------- plain forms

def _to_int8(y):
    """Values that symmetric int8 rows stand for (one scale a row), and the scales."""
    scale = (y.abs().amax(dim=1).double() / 127).float()
    by = torch.where(scale > 0, scale, torch.ones_like(scale)).double()
    q = (y.double() / by[:, None]).round_().clamp_(-127, 127).float()
    return (q * scale[:, None]).to(torch.bfloat16), scale


def _half(raw, at):
    return raw[..., at:at + 2].contiguous().view(torch.float16).float()


def _nibbles(b):
    """[..., 32 low nibbles, 32 high nibbles] of [..., 32 bytes] as one last axis."""
    return torch.cat([b & 15, b >> 4], dim=-1)


def _k_scales(raw):
    """The eight 6-bit scales and mins of a K-quant block's twelve bytes."""
    a, b, c = raw[..., 4:8], raw[..., 8:12], raw[..., 12:16]
    sc = torch.cat([a & 63, (c & 15) | ((a >> 6) << 4)], dim=-1)
    mn = torch.cat([b & 63, (c >> 4) | ((b >> 6) << 4)], dim=-1)
    return sc.float(), mn.float()


def _decode(fmt, raw, rows, cols):
    """f32 weights of the GGUF blocks, each rounded where the format's own decoder rounds."""
    _, be, bb = FORMATS[fmt]
    if fmt == "F32":
        return raw.view(torch.float32).reshape(rows, cols)
    if fmt == "F16":
        return raw.view(torch.float16).float().reshape(rows, cols)
    raw = raw.reshape(rows, cols // be, bb)
    if fmt == "Q8_0":
        w = _half(raw, 0) * raw[..., 2:34].contiguous().view(torch.int8).float()
    elif fmt == "Q4_0":
        w = (_nibbles(raw[..., 2:18]).float() - 8) * _half(raw, 0)
    elif fmt == "Q4_1":
        w = _nibbles(raw[..., 4:20]).float() * _half(raw, 0) + _half(raw, 2)
    elif fmt == "Q5_0":
        bit = torch.arange(8, device=raw.device, dtype=torch.uint8)
        high = ((raw[..., 2:6, None] >> bit) & 1).reshape(rows, -1, 32)
        w = ((_nibbles(raw[..., 6:22]) | (high << 4)).float() - 16) * _half(raw, 0)
    elif fmt in ("Q4_K", "Q5_K"):
        sc, mn = _k_scales(raw)
        nib = raw[..., 48 if fmt == "Q5_K" else 16:].reshape(rows, -1, 4, 32)
        q = _nibbles(nib).reshape(rows, -1, 8, 32)
        if fmt == "Q5_K":
            bit = torch.arange(8, device=raw.device, dtype=torch.uint8)[:, None]
            q = q | (((raw[..., 16:48][..., None, :] >> bit) & 1) << 4)
        w = (_half(raw, 0) * sc)[..., None] * q.float() - (_half(raw, 2) * mn)[..., None]
    else:
        ql = raw[..., :128].reshape(rows, -1, 2, 2, 32)
        qh = raw[..., 128:192].reshape(rows, -1, 2, 1, 32)
        nib = torch.cat([ql & 15, ql >> 4], dim=3)                       # 4 groups of 32 in each half
        shift = torch.arange(0, 8, 2, device=raw.device, dtype=torch.uint8)[:, None]
        q = (nib | (((qh >> shift) & 3) << 4)).reshape(rows, -1, 16, 16)
        sc = raw[..., 192:208].contiguous().view(torch.int8).float()
        w = (_half(raw, 208) * sc)[..., None] * (q.float() - 32)
    return w.reshape(rows, cols)


def _plain(s):
    op = s["op"]
    if op == "gemm":
        k = s["k"]
        y = s["a"][:, :k].float() @ s["w"][:, :k].float().t()
        y = y * s["a_scale"][:, None] * s["w_scale"][None, :]
        return (y + s["b"] if s["bias"] else y).to(DTYPES[s["out"]])
    if op == "weights":
        values, scale = _to_int8(_decode(s["format"], s["raw"], s["rows"], s["cols"]))
        return {"values": values, "scale": scale}
    if op == "norm":
        h = s["x"].float() + s["r"].float() if s["resid"] else s["x"].float()
        y = h * torch.rsqrt(h.square().mean(dim=1, keepdim=True) + 1e-5) * s["w"]
        values, scale = _to_int8(y)
        return {"values": values, "scale": scale, **({"sum": h.to(DTYPES[s["type"]])} if s["resid"] else {})}
    c = s["cols"]
    y = s["gu"][:, :c].float()
    if s["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    elif s["act"] == "gelu":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * y * (1 + 0.044715 * y * y)))
    if s["up"]:
        y = y * s["gu"][:, c:].float()
    values, scale = _to_int8(y)
    return {"values": values, "scale": scale}


# ---------------------------------------------------------------- the library's calls

def _library():
    if "llamini_b200" not in sys.modules:
        spec = importlib.util.spec_from_file_location("llamini_b200", os.path.join(ROOT, "llamini.cpp_b200", "__init__.py"))
        mod = importlib.util.module_from_spec(spec)
        sys.modules["llamini_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["llamini_b200"]


def _own(s):
    lm = _library()
    lib, op, stream = lm.lib(), s["op"], torch.cuda.current_stream().cuda_stream
    if op == "gemm":
        y, b = s["y"], s["b"]
        rc = lib.llamini_gemm_i8_device(
            s["a"].data_ptr(), s["a"].stride(0), s["a_scale"].data_ptr(), s["rows"],
            s["w"].data_ptr(), s["w"].stride(0), s["w_scale"].data_ptr(), s["n"], s["k"],
            b.data_ptr() if b is not None else None, TYPE_IDS[s["out"]], y.data_ptr(), y.stride(0), stream)
        if rc != 0:
            raise RuntimeError(lm.last_error())
        return y
    q, scale, m, c = s["q"], s["scale"], s["rows"], s["cols"]
    if op == "weights":
        rc = lib.llamini_weights_i8_device(FORMATS[s["format"]][0], s["raw"].data_ptr(), m, c,
                                           q.data_ptr(), q.stride(0), scale.data_ptr(), stream)
    elif op == "norm":
        x, r, h = s["x"], s["r"], s["sum"]
        rc = lib.llamini_rms_norm_i8_device(
            TYPE_IDS[s["type"]], x.data_ptr(), x.stride(0), r.data_ptr() if r is not None else None, c,
            h.data_ptr() if h is not None else None, c, s["w"].data_ptr(), 1e-5, m, c,
            q.data_ptr(), q.stride(0), scale.data_ptr(), stream)
    else:
        gu = s["gu"]
        up = gu.data_ptr() + c * gu.element_size() if s["up"] else None
        rc = lib.llamini_glu_i8_device(TYPE_IDS[s["type"]], gu.data_ptr(), gu.stride(0), up, gu.stride(0),
                                       ACTS[s["act"]], m, c, q.data_ptr(), q.stride(0), scale.data_ptr(), stream)
    if rc != 0:
        raise RuntimeError(lm.last_error())
    # the values that the int8 rows stand for
    values = torch.mul(q[:, :c], scale[:, None], out=s["values"])
    return {"values": values, "scale": scale, **({"sum": s["sum"]} if s.get("resid") else {})}


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    if case["op"] == "gemm":
        m, n, k = case["rows"], case["n"], case["k"]
        out = m * n * (4 if case["out"] == "f32" else 2)
        return {"bytes": m * k + n * k + 4 * (m + n) + (4 * n if case["bias"] else 0) + out, "flops": 2 * m * n * k}
    m, c = case["rows"], case["cols"]
    if case["op"] == "weights":
        _, be, bb = FORMATS[case["format"]]
        return {"bytes": m * (c // be * bb + c + 4), "flops": 4 * m * c}
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "norm":
        return {"bytes": m * c * (size * (3 if case["resid"] else 1) + 1) + 4 * (c + m), "flops": 7 * m * c}
    return {"bytes": m * c * (size * (2 if case["up"] else 1) + 1) + 4 * m, "flops": 8 * m * c}


# ---------------------------------------------------------------- 64-bit values

def _exact_int8(y):
    top = y.abs().max(dim=1, keepdim=True).values
    step = top / 127
    q = torch.where(top > 0, torch.round(y / torch.where(top > 0, step, torch.ones_like(step))), torch.zeros_like(y))
    return q * step, step[:, 0]


def _exact_weights(fmt, raw, rows, cols):
    """Element by element through index tables: which byte holds element e of a
    block, at which bit, and which scale it goes by."""
    _, be, bb = FORMATS[fmt]
    if be == 1:
        return raw.view(torch.float32 if bb == 4 else torch.float16).reshape(rows, cols).to(torch.float64)
    blk = raw.reshape(rows * (cols // be), bb)
    half = lambda at: (blk[:, at:at + 2].contiguous().view(torch.float16).to(torch.float64))  # noqa: E731
    at, shift, more, more_shift, group = [], [], [], [], []
    for e in range(be):
        if fmt in ("Q4_0", "Q4_1", "Q5_0"):
            at.append({"Q4_0": 2, "Q4_1": 4, "Q5_0": 6}[fmt] + e % 16)
            shift.append(4 * (e // 16))
            more.append(2 + e // 8)
            more_shift.append(e % 8)
        elif fmt in ("Q4_K", "Q5_K"):
            sub = e // 32
            at.append((16 if fmt == "Q4_K" else 48) + 32 * (sub // 2) + e % 32)
            shift.append(4 * (sub % 2))
            more.append(16 + e % 32)
            more_shift.append(sub)
            group.append(sub)
        elif fmt == "Q6_K":
            part, in_part = divmod(e, 128)
            quarter, lane = divmod(in_part, 32)
            at.append(64 * part + 32 * (quarter % 2) + lane)
            shift.append(4 * (quarter // 2))
            more.append(128 + 32 * part + lane)
            more_shift.append(2 * quarter)
            group.append(e // 16)
        else:
            at.append(2 + e)
            shift.append(0)
    dev = blk.device
    bits = blk[:, torch.tensor(at, device=dev)].to(torch.int32)
    if fmt == "Q8_0":
        w = torch.where(bits > 127, bits - 256, bits).to(torch.float64) * half(0)
        return w.reshape(rows, cols)
    low = (bits >> torch.tensor(shift, device=dev, dtype=torch.int32)) & 15
    del bits
    if fmt in ("Q5_0", "Q5_K", "Q6_K"):
        high = blk[:, torch.tensor(more, device=dev)].to(torch.int32) >> torch.tensor(more_shift, device=dev, dtype=torch.int32)
        low = low + 16 * (high & (3 if fmt == "Q6_K" else 1))
        del high
    q = low.to(torch.float64)
    if fmt == "Q4_0":
        w = half(0) * (q - 8)
    elif fmt == "Q4_1":
        w = half(0) * q + half(2)
    elif fmt == "Q5_0":
        w = half(0) * (q - 16)
    elif fmt == "Q6_K":
        sc = blk[:, 192:208].to(torch.int32)
        sc = torch.where(sc > 127, sc - 256, sc).to(torch.float64) * half(208)
        w = sc[:, torch.tensor(group, device=dev)] * (q - 32)
    else:
        sc, mn = [], []
        b = blk[:, 4:16].to(torch.int32)
        for j in range(8):
            if j < 4:
                sc.append(b[:, j] % 64)
                mn.append(b[:, j + 4] % 64)
            else:
                sc.append(b[:, j + 4] % 16 + 16 * (b[:, j - 4] // 64))
                mn.append(b[:, j + 4] // 16 + 16 * (b[:, j] // 64))
        g = torch.tensor(group, device=dev)
        w = half(0) * torch.stack(sc, 1).to(torch.float64)[:, g] * q - half(2) * torch.stack(mn, 1).to(torch.float64)[:, g]
    return w.reshape(rows, cols)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "gemm":
        k = case["k"]
        a = s["a"][:, :k].to(torch.float64) * s["a_scale"].to(torch.float64).unsqueeze(1)
        w = s["w"][:, :k].to(torch.float64) * s["w_scale"].to(torch.float64).unsqueeze(1)
        y = torch.einsum("mk,nk->mn", a, w)
        return y + s["b"].to(torch.float64) if case["bias"] else y
    if op == "weights":
        values, scale = _exact_int8(_exact_weights(case["format"], s["raw"], case["rows"], case["cols"]))
        return {"values": values, "scale": scale}
    if op == "norm":
        h = s["x"].to(torch.float64)
        if case["resid"]:
            h = h + s["r"].to(torch.float64)
        rms = torch.sqrt((h * h).sum(dim=1) / case["cols"] + 1e-5)
        values, scale = _exact_int8(h / rms.unsqueeze(1) * s["w"].to(torch.float64))
        return {"values": values, "scale": scale, **({"sum": h} if case["resid"] else {})}
    gate, c = s["gu"][:, :case["cols"]].to(torch.float64), case["cols"]
    if case["act"] == "silu":
        gate = gate * torch.sigmoid(gate)
    elif case["act"] == "gelu":
        inner = math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3)
        gate = gate * torch.sigmoid(2 * inner)      # (1 + tanh z) / 2 = sigmoid(2 z)
    values, scale = _exact_int8(gate * s["gu"][:, c:].to(torch.float64) if case["up"] else gate)
    return {"values": values, "scale": scale}
