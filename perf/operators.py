"""The 8-bit feed-forward operators: RMS norm with the residual's addition and an 8-bit output, the gated unit with an
8-bit output, and the product of 8-bit floating point operands with a scale for each block of 128.

`listed()` holds the fixed cases, `draw()` makes more of the same ranges, `prepare()` makes a case's inputs and buffers
on the GPU, `run()` is one pass, in plain 32-bit torch operations or, where `own` is set, through h3metal_amd.ops;
`exact()` gives the same outputs in 64 bits.
"""

import math

import torch

own = False
DEV = "cuda"
BLOCK = 128      # columns that share a scale
F8_MAX = 448.0   # the largest e4m3 value
EPS = 1e-6
F8 = torch.float8_e4m3fn
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8, "u8": torch.uint8, "f8": F8}


# -- the cases ------------------------------------------------------------------------------------------------------

def listed():
    return [
        # One row of a text model's residual stream: what counts is the latency of the call.
        dict(name="norm_token", op="norm", M=1, D=4096, x="bf16", res="bf16", weight=True),
        # A prompt of 301 rows, a width whose last block is short, half precision.
        dict(name="norm_text", op="norm", M=301, D=2632, x="f16", res="f16", weight=True),
        # Joint text + image rows of a 2048 x 2048 image into a float residual stream: bound by memory.
        dict(name="norm_2048", op="norm", M=16896, D=4096, x="bf16", res="f32", weight=True),
        # The gated unit of one token, and of a 2048 x 2048 image's rows.
        dict(name="swiglu_token", op="swiglu", M=1, D=10240, x="bf16"),
        dict(name="swiglu_2048", op="swiglu", M=16896, D=10240, x="bf16"),
        # The products of one token: all of the time is the reading of the weights.
        dict(name="gemm_token", op="gemm", M=1, N=4096, K=4096, epi=0, out="bf16", bias=False),
        # Nine rows, odd columns, a short last block of K, float outputs with a bias.
        dict(name="gemm_ragged", op="gemm", M=9, N=1001, K=2000, epi=0, out="f32", bias=True),
        # A text encoder's projection of a prompt of 300 rows.
        dict(name="gemm_text", op="gemm", M=300, N=4096, K=4096, epi=0, out="f16", bias=False),
        # The qkv projection of a 2048 x 2048 image: bound by the matrix units, the largest case here.
        dict(name="gemm_qkv_2048", op="gemm", M=16896, N=12288, K=4096, epi=0, out="bf16", bias=False),
        # The second product of the feed-forward part at 1024 x 1024, into the gated float residual.
        dict(name="gemm_residual_1024", op="gemm", M=4608, N=4096, K=10240, epi=1, out="f32", bias=False),
        # The norm with int8 rows in front of the int8 projection that takes them.
        dict(name="norm_q8_gemm", op="norm_gemm", M=1024, D=4096, N=4096),
        # The feed-forward part of a block at 1024 x 1024: norm, product, gated unit, product.
        dict(name="mlp_1024", op="mlp", M=4608, D=4096, F=10240),
    ]


LARGEST = 2.0 * 16896 * 12288 * 4096  # operations of the largest listed product


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "swiglu", "swiglu", "gemm", "gemm", "gemm", "gemm", "norm_gemm", "mlp"])
    if kind in ("norm", "swiglu"):
        M = _log(rng, 1, 16896)
        D = _log(rng, 64, 10240)  # any width
        if rng.random() < 0.6:    # most widths are whole blocks
            D = max(BLOCK, D // BLOCK * BLOCK)
        x = rng.choice(["bf16", "bf16", "f16", "f32"])
        if kind == "swiglu":
            return dict(op=kind, M=M, D=D, x=x)
        return dict(op=kind, M=M, D=D, x=x, res=rng.choice(["none", "f32", x]), weight=rng.random() < 0.8)
    if kind == "gemm":
        while True:
            M, N, K = _log(rng, 1, 16896), _log(rng, 32, 12288), 16 * _log(rng, 4, 768)
            if rng.random() < 0.6:
                N, K = max(BLOCK, N // BLOCK * BLOCK), max(BLOCK, K // BLOCK * BLOCK)
            if 2.0 * M * N * K <= LARGEST:
                break
        epi = rng.choice([0, 0, 0, 1])
        return dict(op=kind, M=M, N=N, K=K, epi=epi, out="f32" if epi else rng.choice(["bf16", "f16", "f32"]),
                    bias=rng.random() < 0.3)
    if kind == "norm_gemm":
        return dict(op=kind, M=_log(rng, 1, 8192), D=64 * _log(rng, 8, 80), N=BLOCK * _log(rng, 4, 64))
    return dict(op="mlp", M=_log(rng, 1, 4608), D=BLOCK * _log(rng, 8, 32), F=BLOCK * _log(rng, 16, 80))


# -- inputs ---------------------------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _rows(g, M, D, dtype):
    """Activations: normal, a few of the columns larger."""
    x = _normal(g, M, D)
    x[:, torch.randperm(D, generator=g, device=DEV)[:max(1, D // 64)]] *= 8
    return x.to(TYPES[dtype])


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _pad(x, rows, cols):
    return torch.nn.functional.pad(x, (0, cols - x.shape[1], 0, rows - x.shape[0]))


def _made_codes(x):
    """Activations as a producer leaves them: codes and a scale for each row and block of columns."""
    M, K = x.shape
    b = _pad(x, M, _blocks(K) * BLOCK).view(M, -1, BLOCK)
    s = b.abs().amax(-1) / F8_MAX
    q = (b / s[..., None]).clamp(-F8_MAX, F8_MAX).view(M, -1)[:, :K]
    return q.to(F8).contiguous(), s


def _made_weight(g, N, K):
    """A weight of variance 1 / K: codes and a scale for each block of 128 rows x 128 columns."""
    nb, kb = _blocks(N), _blocks(K)
    w = _pad(_normal(g, N, K) / math.sqrt(K), nb * BLOCK, kb * BLOCK).view(nb, BLOCK, kb, BLOCK)
    s = w.abs().amax((1, 3)) / F8_MAX
    q = (w / s[:, None, :, None]).clamp(-F8_MAX, F8_MAX).view(nb * BLOCK, kb * BLOCK)[:N, :K]
    return q.to(F8).contiguous(), s


def _inputs(c, seed):
    g, op, M = _gen(seed), c["op"], c["M"]
    if op == "norm":
        return dict(x=_rows(g, M, c["D"], c["x"]), res=None if c["res"] == "none" else _rows(g, M, c["D"], c["res"]),
                    w=1 + 0.1 * _normal(g, c["D"]) if c["weight"] else None)
    if op == "swiglu":
        return dict(x=(2 * _normal(g, M, 2 * c["D"])).to(TYPES[c["x"]]))
    if op == "gemm":
        d = dict(zip(("a", "sa"), _made_codes(_rows(g, M, c["K"], "f32"))))
        d.update(zip(("w", "sw"), _made_weight(g, c["N"], c["K"])))
        if c["bias"]:
            d["bias"] = _normal(g, c["N"])
        if c["epi"]:  # the residual stream, the rows' modality (text, image) and its gates
            d.update(x=_normal(g, M, c["N"]), rtype=(torch.arange(M, device=DEV) >= M // 8).to(torch.uint8),
                     gate=1 + 0.1 * _normal(g, 2, c["N"]))
        return d
    if op == "norm_gemm":
        return dict(x=_rows(g, M, c["D"], "bf16"), res=_rows(g, M, c["D"], "bf16"), w=1 + 0.1 * _normal(g, c["D"]),
                    wq=torch.randint(-127, 128, (c["N"], c["D"]), generator=g, device=DEV, dtype=torch.int8),
                    sw=torch.rand(c["N"], generator=g, device=DEV) * 1e-4 + 1e-4)
    D, F = c["D"], c["F"]
    d = dict(x=_rows(g, M, D, "bf16"), res=_rows(g, M, D, "bf16"), w=1 + 0.1 * _normal(g, D))
    d.update(zip(("w1", "s1"), _made_weight(g, 2 * F, D)))
    d.update(zip(("w2", "s2"), _made_weight(g, D, F)))
    return d


# -- the framework's buffers (reached where `own` is set) -------------------------------------------------------------

_gpu = None


def _context():
    """The program's device context."""
    global _gpu
    if _gpu is None:
        from h3metal_amd.gpu import Gpu
        _gpu = Gpu()
    return _gpu


class _Device:
    """What torch makes a tensor from; it keeps the buffer as long as the tensor lives."""

    def __init__(self, ptr, t, typestr):
        self.buf = t.buf
        self.__cuda_array_interface__ = dict(shape=tuple(t.shape), typestr=typestr, data=(ptr, False), version=2)


def _view(t):
    """A torch tensor over the device memory of a framework tensor."""
    from h3metal_amd.gpu import lib
    raw = {"f32": "<f4", "f16": "<f2", "bf16": "<i2", "i8": "|i1", "u8": "|u1", "f8": "|u1"}[t.dtype]
    x = torch.as_tensor(_Device(lib().h3_buffer_device(t.buf.handle) + t.offset, t, raw), device=DEV)
    return x.view(TYPES[t.dtype]) if t.dtype in ("bf16", "f8") else x


def _held(x):
    """`x` in a buffer of the framework."""
    if x is None:
        return None
    dtype = next(n for n, t in TYPES.items() if t == x.dtype)
    t = _context().empty(x.shape, dtype)
    bits = torch.uint8 if dtype == "f8" else x.dtype
    _view(t).view(bits).copy_(x.view(bits))
    return t


def _own_state(c, d):
    from h3metal_amd import ops
    new, op, M = _context().empty, c["op"], c["M"]
    s = {n: _held(x) for n, x in d.items()}
    if op == "norm":
        s.update(o=new((M, c["D"]), "f8"), so=new((M, _blocks(c["D"])), "f32"))
        s["ro"] = new((M, c["D"]), c["res"]) if c["res"] != "none" else None
        s["back"] = [_view(s[n]) for n in ("o", "so") + (("ro",) if s["ro"] else ())]
    elif op == "swiglu":
        s.update(o=new((M, c["D"]), "f8"), so=new((M, _blocks(c["D"])), "f32"))
        s["back"] = [_view(s["o"]), _view(s["so"])]
    elif op == "gemm":
        s["weight"] = ops.QWeight("f8", s["w"], s["sw"], c["N"], c["K"], bias=s.get("bias"))
        s["o"] = s["x"] if c["epi"] else new((M, c["N"]), c["out"])
        s["back"] = [_view(s["o"])]
    elif op == "norm_gemm":
        rows = ops.pad_rows(M, 64)  # int8 products take rows padded to the default tile's height
        s["weight"] = ops.QWeight("q8", s["wq"], s["sw"], c["N"], c["D"])
        s.update(ro=new((M, c["D"]), "bf16"), a=new((rows, c["D"]), "i8"), sa=new((rows,), "f32"),
                 o=new((rows, c["N"]), "bf16"))
        s["back"] = [_view(s["ro"]), _view(s["sa"])[:M], _view(s["o"])[:M]]
    else:
        D, F = c["D"], c["F"]
        s["up"], s["down"] = ops.QWeight("f8", s["w1"], s["s1"], 2 * F, D), ops.QWeight("f8", s["w2"], s["s2"], D, F)
        s.update(ro=new((M, D), "bf16"), a=new((M, D), "f8"), sa=new((M, _blocks(D)), "f32"),
                 h=new((M, 2 * F), "bf16"), b=new((M, F), "f8"), sb=new((M, _blocks(F)), "f32"), o=new((M, D), "bf16"))
        s["back"] = [_view(s["ro"]), _view(s["o"])]
    return s


def prepare(case, seed):
    d = _inputs(case, seed)
    s = _own_state(case, d) if own else d
    s["case"] = case
    torch.cuda.synchronize()
    return s


# -- one pass in plain operations -------------------------------------------------------------------------------------

def _added(x, res):
    """The residual's sum, rounded once to its type."""
    return x if res is None else (res.float() + x.float()).to(res.dtype)


def _normed(h, w):
    t = h.float()
    t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS)
    return t if w is None else t * w


def _codes(v):
    """e4m3 codes of the rows of v and a scale for each block of 128 columns."""
    M, D = v.shape
    b = _pad(v, M, _blocks(D) * BLOCK).view(M, -1, BLOCK)
    amax = b.abs().amax(-1)
    s = torch.where(amax > 0, amax / F8_MAX, torch.ones_like(amax))
    q = (b / s[..., None]).clamp(-F8_MAX, F8_MAX).view(M, -1)[:, :D]
    return q.to(F8).contiguous(), s


def _gated(x):
    v, g = x.float().chunk(2, -1)
    return v * (g / (1 + torch.exp(-g)))


def _product(a, sa, w, sw):
    x = a.float() * sa.repeat_interleave(BLOCK, 1)[:, :a.shape[1]]
    y = w.float() * sw.repeat_interleave(BLOCK, 0)[:w.shape[0]].repeat_interleave(BLOCK, 1)[:, :w.shape[1]]
    return x @ y.t()


def _plain(c, s):
    op = c["op"]
    if op == "norm":
        h = _added(s["x"], s["res"])
        return list(_codes(_normed(h, s["w"]))) + ([h] if s["res"] is not None else [])
    if op == "swiglu":
        return list(_codes(_gated(s["x"])))
    if op == "gemm":
        v = _product(s["a"], s["sa"], s["w"], s["sw"])
        if c["bias"]:
            v = v + s["bias"]
        if c["epi"]:
            return [s["x"].add_(s["gate"][s["rtype"].long()] * v)]
        return [v.to(TYPES[c["out"]])]
    h = _added(s["x"], s["res"])
    v = _normed(h, s["w"])
    if op == "norm_gemm":
        amax = v.abs().amax(-1, keepdim=True)
        sa = torch.where(amax > 0, amax / 127, torch.ones_like(amax))
        out = (torch.round(v / sa) @ s["wq"].float().t()) * sa * s["sw"]
        return [h, sa[:, 0].contiguous(), out.to(torch.bfloat16)]
    up = _product(*_codes(v), s["w1"], s["s1"]).to(torch.bfloat16)
    return [h, _product(*_codes(_gated(up)), s["w2"], s["s2"]).to(torch.bfloat16)]


# -- one pass of either ------------------------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    if not own:
        return _plain(c, s)
    from h3metal_amd import ops
    g, op, M = _context(), c["op"], c["M"]
    if op == "norm":
        ops.rms_norm_q8(g, s["x"], s["w"], s["o"], s["so"], M, c["D"], eps=EPS, res=s["res"], res_out=s["ro"])
    elif op == "swiglu":
        ops.swiglu_f8(g, s["x"], s["o"], s["so"], M, c["D"])
    elif op == "gemm":
        ops.gemm(g, s["a"], s["weight"], s["o"], M, sa=s["sa"], epi=c["epi"], rtype=s.get("rtype"), gate=s.get("gate"))
    elif op == "norm_gemm":
        ops.rms_norm_q8(g, s["x"], s["w"], s["a"], s["sa"], M, c["D"], eps=EPS, res=s["res"], res_out=s["ro"])
        ops.gemm(g, s["a"], s["weight"], s["o"], M, sa=s["sa"])
    else:
        ops.rms_norm_q8(g, s["x"], s["w"], s["a"], s["sa"], M, c["D"], eps=EPS, res=s["res"], res_out=s["ro"])
        ops.gemm(g, s["a"], s["up"], s["h"], M, sa=s["sa"])
        ops.swiglu_f8(g, s["h"], s["b"], s["sb"], M, c["F"])
        ops.gemm(g, s["b"], s["down"], s["o"], M, sa=s["sb"])
    return s["back"]


# -- what a pass cannot do without ------------------------------------------------------------------------------------

SIZE = {"f32": 4, "f16": 2, "bf16": 2, "none": 0}


def _norm_bytes(M, D, x, res, weight, scales):
    return M * D * (SIZE[x] + 2 * SIZE[res] + 1) + 4 * M * scales + (4 * D if weight else 0)


def _swiglu_bytes(M, D, x):
    return M * D * (2 * SIZE[x] + 1) + 4 * M * _blocks(D)


def _gemm_work(M, N, K, out, epi=0, bias=False):
    scales = 4 * _blocks(K) * (M + _blocks(N))
    more = (4 * N if bias else 0) + (M * N * SIZE[out] + M + 8 * N if epi else 0)
    return M * K + N * K + scales + M * N * SIZE[out] + more, 2.0 * M * N * K


def work(case):
    c, op, M = case, case["op"], case["M"]
    if op == "norm":
        b, f = _norm_bytes(M, c["D"], c["x"], c["res"], c["weight"], _blocks(c["D"])), 6.0 * M * c["D"]
    elif op == "swiglu":
        b, f = _swiglu_bytes(M, c["D"], c["x"]), 8.0 * M * c["D"]
    elif op == "gemm":
        b, f = _gemm_work(M, c["N"], c["K"], c["out"], c["epi"], c["bias"])
    elif op == "norm_gemm":  # the codes stay on the chip at best
        D, N = c["D"], c["N"]
        b, f = M * D * 6 + 4 * D + 4 * M + N * D + 4 * N + M * N * 2, 2.0 * M * N * D
    else:
        D, F = c["D"], c["F"]
        up, down = _gemm_work(M, 2 * F, D, "bf16"), _gemm_work(M, D, F, "bf16")
        b = _norm_bytes(M, D, "bf16", "bf16", True, _blocks(D)) + up[0] + _swiglu_bytes(M, F, "bf16") + down[0]
        f = up[1] + down[1]
    return dict(bytes=float(b), flops=float(f))


# -- the same in 64 bits ----------------------------------------------------------------------------------------------

def _e4m3(x):
    """x in float64, rounded to the nearest e4m3 value (half to even), the largest ones kept at 448."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-F8_MAX, F8_MAX)


def _by_block(v, f):
    """f(block) for each block of 128 columns: what it gives side by side."""
    return [torch.cat(p, 1) for p in zip(*(f(v[:, k:k + BLOCK]) for k in range(0, v.shape[1], BLOCK)))]


def _exact_block(v):
    top = v.abs().max(1, keepdim=True).values
    s = torch.where(top > 0, top / F8_MAX, 1.0)
    return _e4m3(v / s), s


def _exact_norm(d):
    h = d["x"].double()
    if d["res"] is not None:
        h = (h + d["res"].double()).to(d["res"].dtype).double()
    v = h * torch.rsqrt(h.square().sum(1, keepdim=True) / h.shape[1] + EPS)
    return h, v * d["w"].double() if d["w"] is not None else v


def _exact_gate(x):
    x = x.double()
    n = x.shape[1] // 2
    return x[:, :n] * x[:, n:] * torch.sigmoid(x[:, n:])


def _exact_product(a, sa, w, sw):
    a, w, sa, sw = a.double(), w.double().t().contiguous(), sa.double(), sw.double()
    v = torch.zeros(a.shape[0], w.shape[1], device=DEV, dtype=torch.float64)
    col = torch.arange(w.shape[1], device=DEV) // BLOCK
    for b in range(sa.shape[1]):  # block by block: its sum times its two scales
        part = slice(b * BLOCK, (b + 1) * BLOCK)
        v += (a[:, part] @ w[part]) * sa[:, b:b + 1] * sw[col, b]
    return v


def exact(case, seed):
    c, op, d = case, case["op"], _inputs(case, seed)
    if op == "norm":
        h, v = _exact_norm(d)
        return _by_block(v, _exact_block) + ([h] if d["res"] is not None else [])
    if op == "swiglu":
        return _by_block(_exact_gate(d["x"]), _exact_block)
    if op == "gemm":
        v = _exact_product(d["a"], d["sa"], d["w"], d["sw"])
        if c["bias"]:
            v += d["bias"].double()
        return [d["x"].double() + d["gate"].double()[d["rtype"].long()] * v if c["epi"] else v]
    h, v = _exact_norm(d)
    if op == "norm_gemm":
        top = v.abs().max(1, keepdim=True).values
        s = torch.where(top > 0, top / 127, 1.0)
        return [h, s[:, 0], (torch.round(v / s) @ d["wq"].double().t()) * s * d["sw"].double()]
    up = _exact_product(*_by_block(v, _exact_block), d["w1"], d["s1"]).to(torch.bfloat16)
    return [h, _exact_product(*_by_block(_exact_gate(up), _exact_block), d["w2"], d["s2"])]
