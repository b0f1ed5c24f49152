"""The text model's operators over a paged cache of keys and values: the per-head norm and rotary embedding of queries and
keys, written to rows and to the cache's pages, and the attention of a batch's new tokens over those pages.

`listed()` holds the fixed cases, `draw()` makes more of the same ranges, `prepare()` makes a case's inputs and buffers
on the GPU, `run()` is one pass, in plain 32-bit torch operations or, where `own` is set, through h3metal_amd.ops;
`exact()` gives the same outputs in 64 bits.

A case's batch has B sequences with `new_lo` to `new_hi` new tokens each, behind `old_lo` to `old_hi` tokens that the cache
holds already; the lengths come from the number `lens` alone.
"""

import math
import random

import torch

own = False
DEV = "cuda"
EPS = 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i32": torch.int32}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BASE = 1e6           # of the rotary frequencies
TRAINED = 32768      # positions that the unscaled frequencies were made for
FAR = 900_000        # first rotary position of the cases with positions of their own


# -- the cases ------------------------------------------------------------------------------------------------------

def _batch(B, new_lo, new_hi, old_lo, old_hi, page, lens):
    return dict(B=B, new_lo=new_lo, new_hi=new_hi, old_lo=old_lo, old_hi=old_hi, page=page, lens=lens)


def _heads(H, KVH, D, dtype):
    return dict(H=H, KVH=KVH, D=D, dtype=dtype)


def _rotary(x, rot, norm, inter, scaling, far):
    return dict(x=x, rot=rot, norm=norm, inter=inter, scaling=scaling, far=far)


def listed():
    return [
        # One new token of one text: what counts is the latency of the call.
        dict(name="rope_token", op="rope", **_batch(1, 1, 1, 511, 511, 16, 1), **_heads(32, 8, 128, "bf16"),
             **_rotary("bf16", 128, True, False, "none", False)),
        # Five prompts of uneven length from float rows into a half-precision cache, a part of the head rotated, pairs side by
        # side, positions of their own far out.
        dict(name="rope_ragged", op="rope", **_batch(5, 17, 141, 0, 300, 32, 2), **_heads(16, 4, 64, "f16"),
             **_rotary("f32", 40, False, True, "linear", True)),
        # A chunk of a long document's rows, frequencies scaled for its length.
        dict(name="rope_chunk", op="rope", **_batch(1, 8192, 8192, 57344, 57344, 64, 3), **_heads(32, 8, 128, "bf16"),
             **_rotary("bf16", 128, True, False, "yarn", False)),
        # One new token of one short text.
        dict(name="attn_token", op="attn", **_batch(1, 1, 1, 511, 511, 16, 4), **_heads(32, 8, 128, "bf16"), causal=True),
        # One new token of each of 64 texts of uneven length: bound by the reading of the cache.
        dict(name="attn_tokens_64", op="attn", **_batch(64, 1, 1, 64, 8191, 16, 5), **_heads(32, 8, 128, "bf16"),
             causal=True),
        # One new token of one long text: the same keys have to be spread over the whole chip.
        dict(name="attn_token_long", op="attn", **_batch(1, 1, 1, 131071, 131071, 64, 6), **_heads(32, 8, 128, "bf16"),
             causal=True),
        # A chunk of 512 tokens behind a long prefix.
        dict(name="attn_chunk", op="attn", **_batch(1, 512, 512, 15872, 15872, 16, 7), **_heads(32, 8, 128, "bf16"),
             causal=True),
        # A text encoder's batch of prompts behind a shared template's rows, half precision.
        dict(name="attn_prompts", op="attn", **_batch(8, 40, 512, 24, 24, 16, 8), **_heads(32, 8, 128, "f16"), causal=True),
        # Image rows that look at all of a cached text, heads of 96 channels with keys of their own, odd lengths.
        dict(name="attn_cross_96", op="attn", **_batch(3, 333, 1037, 0, 700, 32, 9), **_heads(16, 16, 96, "f16"),
             causal=False),
        # A prompt of 8192 tokens: bound by the matrix units, the largest case here.
        dict(name="attn_prompt_8192", op="attn", **_batch(1, 8192, 8192, 0, 0, 64, 10), **_heads(32, 8, 128, "bf16"),
             causal=True),
        # A serving step of a layer: chunks and single tokens in one batch, the cache's update and the attention over it.
        dict(name="layer_mixed", op="layer", **_batch(24, 1, 96, 200, 4000, 16, 11), **_heads(32, 8, 128, "bf16"),
             **_rotary("bf16", 128, True, False, "none", False), causal=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


LARGEST = 8192 * 8193 / 2 * 4 * 32 * 128  # operations of the largest listed case
MOST_KEYS = 64 * 8192                     # keys of all sequences
MOST_ROWS = 8192                          # new tokens of all sequences


def draw(rng):
    op = rng.choice(["rope", "rope", "attn", "attn", "attn", "layer"])
    while True:
        D = rng.choice([128, 128, 64, 96])
        KVH = rng.choice([1, 2, 4, 8, 8])
        H = min(64, KVH * rng.choice([1, 2, 4, 4, 5, 8]))
        kind = rng.choice(["one", "tokens", "tokens", "prompts", "chunk", "mixed"])
        if kind == "one":
            old = _log(rng, 1, 131072) - 1
            b = (1, 1, 1, old, old)
        elif kind == "tokens":
            lo = _log(rng, 1, 4096)
            b = (_log(rng, 2, 128), 1, 1, lo, _log(rng, lo, 8192))
        elif kind == "prompts":
            lo = _log(rng, 1, 512)
            b = (_log(rng, 1, 16), lo, _log(rng, lo, 2048), 0, rng.choice([0, 24, 100]))
        elif kind == "chunk":
            n, old = _log(rng, 2, 8192), _log(rng, 1, 65536)
            b = (1, n, n, old, old)
        else:
            lo = _log(rng, 1, 2000)
            b = (_log(rng, 2, 48), 1, _log(rng, 2, 128), lo, _log(rng, lo, 6000))
        c = dict(op=op, **_batch(*b, rng.choice([16, 16, 32, 64, 128, 256]), rng.randrange(1 << 20)),
                 **_heads(H, KVH, D, rng.choice(["bf16", "bf16", "f16"])))
        if op != "attn":
            rot = rng.choice([D, D, D // 2, 2 * rng.randrange(1, D // 2)])
            c.update(_rotary(rng.choice([c["dtype"], c["dtype"], "f32"]), rot, rng.random() < 0.7, rng.random() < 0.4,
                             rng.choice(["none", "linear", "ntk", "yarn"]), rng.random() < 0.3))
        if op != "rope":
            c["causal"] = rng.random() < 0.8
        new, keys = lengths(c)
        if sum(new) <= MOST_ROWS and sum(keys) <= MOST_KEYS and (op == "rope" or _pairs(c) * 4 * H * D <= LARGEST):
            return c


def lengths(c):
    """New tokens and keys (old and new) of each sequence."""
    rng = random.Random(c["lens"])
    new = [rng.randint(c["new_lo"], c["new_hi"]) for _ in range(c["B"])]
    return new, [n + rng.randint(c["old_lo"], c["old_hi"]) for n in new]


def _pairs(c):
    """(query, key) pairs of one head that see each other."""
    return sum(n * L - (n * (n - 1) // 2 if c["causal"] else 0) for n, L in zip(*lengths(c)))


# -- inputs ---------------------------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _inputs(c, seed):
    g = _gen(seed)
    H, KVH, D, page, dtype = c["H"], c["KVH"], c["D"], c["page"], TYPES[c["dtype"]]
    new, keys = lengths(c)
    M, need = sum(new), [-(-L // page) for L in keys]
    pages = sum(need) + 3  # a few pages belong to nobody
    d = dict(q_start=torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], device=DEV, dtype=torch.int32),
             kv_len=torch.tensor(keys, device=DEV, dtype=torch.int32))
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)  # pages were given out in no order
    table, at = torch.zeros(len(keys), max(need), device=DEV, dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n], at = order[at:at + n], at + n
    d["table"] = table
    for name in ("kc", "vc"):
        t = torch.empty(pages, KVH, page, D, device=DEV, dtype=dtype)
        for i in range(0, pages, 1024):
            t[i:i + 1024] = _normal(g, *t[i:i + 1024].shape).to(dtype)
        d[name] = t
    if c["op"] == "attn":
        d["q"] = _normal(g, M, H * D).to(dtype)
        return d
    x = _normal(g, M, H + 2 * KVH, D)
    x[:, :H + KVH, :max(1, D // 32)] *= 8  # a few of the channels are larger before the norm
    d["qkv"] = x.view(M, -1).to(TYPES[c["x"]])
    if c["norm"]:
        d["wq"], d["wk"] = 1 + 0.1 * _normal(g, D), 1 + 0.1 * _normal(g, D)
    if c["far"]:
        first = torch.randint(0, 1000, (len(keys),), generator=g, device=DEV) + FAR
        d["pos"] = torch.cat([first[b] + torch.arange(n, device=DEV) for b, n in enumerate(new)]).to(torch.int32)
    return d


# -- rotary frequencies ------------------------------------------------------------------------------------------------

FACTOR = 4.0  # by which the scaled kinds lengthen the context


def _frequencies(rot, scaling):
    """Radians per position of each pair in 64 bits, and the factor on rotated channels."""
    i = torch.arange(rot // 2, device=DEV, dtype=torch.float64)
    base = BASE * FACTOR ** (rot / (rot - 2)) if scaling == "ntk" and rot > 2 else BASE
    f = base ** (-2 * i / rot)
    if scaling == "linear":
        return f / FACTOR, 1.0
    if scaling != "yarn":
        return f, 1.0

    def pair(turns):  # the pair that turns so often over the trained positions
        return rot * math.log(TRAINED / (turns * 2 * math.pi)) / (2 * math.log(BASE))

    lo, hi = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), rot // 2 - 1)
    ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
    return f * (1 - ramp) + f / FACTOR * ramp, 0.1 * math.log(FACTOR) + 1.0


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
    raw = {"f32": "<f4", "f16": "<f2", "bf16": "<i2", "i32": "<i4"}[t.dtype]
    x = torch.as_tensor(_Device(lib().h3_buffer_device(t.buf.handle) + t.offset, t, raw), device=DEV)
    return x.view(torch.bfloat16) if t.dtype == "bf16" else x


def _held(x):
    """`x` in a buffer of the framework."""
    t = _context().empty(x.shape, next(n for n, k in TYPES.items() if k == x.dtype))
    _view(t).copy_(x)
    return t


def _own_state(c, d):
    s = {n: _held(x) for n, x in d.items()}
    M, op = sum(lengths(c)[0]), c["op"]
    if op != "attn":
        from h3metal_amd import rope
        freq, s["rope_scale"] = rope.frequencies(c["rot"], base=BASE, scaling=c["scaling"], factor=FACTOR, trained=TRAINED)
        s["turns"] = _context().upload(rope.turns(freq), "u32")
        s["q"] = _context().empty((M, c["H"] * c["D"]), c["dtype"])
    if op != "rope":
        s["o"] = _context().empty((M, c["H"] * c["D"]), c["dtype"])
    s["back"] = [_view(s[n]) for n in {"rope": ("q", "kc", "vc"), "attn": ("o",), "layer": ("o", "kc", "vc")}[op]]
    return s


def prepare(case, seed):
    d = _inputs(case, seed)
    s = _own_state(case, d) if own else d
    if case["op"] != "attn" and not own:
        s["freq"], s["factor"] = _frequencies(case["rot"], case["scaling"])
    s["case"], s["M"] = case, sum(lengths(case)[0])
    s["max_q"], s["max_kv"] = max(lengths(case)[0]), max(lengths(case)[1])
    torch.cuda.synchronize()
    return s


# -- one pass in plain operations -------------------------------------------------------------------------------------

def _rows(c, s):
    """Each new row's sequence and place in the cache."""
    row = torch.arange(s["M"], device=DEV)
    b = torch.searchsorted(s["q_start"].long(), row, right=True) - 1
    return b, s["kv_len"].long()[b] - s["q_start"].long()[b + 1] + row


def _rotated(v, angle, inter, factor):
    n = angle.shape[-1]
    cos, sin = (torch.cos(angle) * factor).float()[:, None], (torch.sin(angle) * factor).float()[:, None]
    a, b = (v[..., 0:2 * n:2], v[..., 1:2 * n:2]) if inter else (v[..., :n], v[..., n:2 * n])
    x, y = a * cos - b * sin, b * cos + a * sin
    return torch.cat([torch.stack([x, y], -1).flatten(-2) if inter else torch.cat([x, y], -1), v[..., 2 * n:]], -1)


def _plain_rope(c, s):
    H, KVH, D, dtype = c["H"], c["KVH"], c["D"], TYPES[c["dtype"]]
    x = s["qkv"].view(s["M"], H + 2 * KVH, D).float()
    b, at = _rows(c, s)
    angle = (s["pos"] if c["far"] else at).double()[:, None] * s["freq"]

    def side(v, w):
        if c["norm"]:
            v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * w
        return _rotated(v, angle, c["inter"], s["factor"]).to(dtype)

    page = s["table"].long()[b, at // c["page"]]
    s["kc"][page, :, at % c["page"]] = side(x[:, H:H + KVH], s.get("wk"))
    s["vc"][page, :, at % c["page"]] = x[:, H + KVH:].to(dtype)
    return side(x[:, :H], s.get("wq")).reshape(s["M"], H * D)


def _plain_attention(c, s, q):
    H, KVH, D, page = c["H"], c["KVH"], c["D"], c["page"]
    out, m = torch.empty(s["M"], H * D, device=DEV, dtype=q.dtype), 0
    for b, (n, L) in enumerate(zip(*lengths(c))):
        pages = s["table"][b, :-(-L // page)].long()
        last = torch.arange(L - n, L, device=DEV) if c["causal"] else torch.full((n,), L - 1, device=DEV)
        hidden = (torch.arange(L, device=DEV) > last[:, None]).repeat_interleave(H // KVH, 0)
        for h in range(KVH):
            k, v = (s[t][pages, h].reshape(-1, D)[:L].float() for t in ("kc", "vc"))
            x = q[m:m + n].view(n, KVH, -1, D)[:, h].reshape(-1, D).float() @ k.t() * D ** -0.5
            x.masked_fill_(hidden, -math.inf)
            x = torch.exp(x - x.amax(-1, keepdim=True))
            o = (x @ v) / x.sum(-1, keepdim=True)
            out[m:m + n].view(n, KVH, -1, D)[:, h] = o.view(n, -1, D).to(out.dtype)
        m += n
    return out


def _plain(c, s):
    if c["op"] == "attn":
        return [_plain_attention(c, s, s["q"])]
    q = _plain_rope(c, s)
    return [q if c["op"] == "rope" else _plain_attention(c, s, q), s["kc"], s["vc"]]


# -- one pass of either ------------------------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    if not own:
        return _plain(c, s)
    from h3metal_amd import ops
    g, D = _context(), c["D"]
    if c["op"] != "attn":
        ops.qk_norm_rope_paged(g, s["qkv"], s.get("wq"), s.get("wk"), s["turns"], s["q"], s["kc"], s["vc"], s["table"],
                               s["q_start"], s["kv_len"], M=s["M"], B=c["B"], Hq=c["H"], Hk=c["KVH"], hd=D, rot=c["rot"],
                               eps=EPS, norm=c["norm"], interleaved=c["inter"], rope_scale=s["rope_scale"],
                               pos=s.get("pos"))
    if c["op"] != "rope":
        ops.attention_paged(g, s["q"], s["kc"], s["vc"], s["o"], s["table"], s["q_start"], s["kv_len"], M=s["M"], B=c["B"],
                            H=c["H"], KVH=c["KVH"], D=D, scale=D ** -0.5, causal=c["causal"], max_q=s["max_q"],
                            max_kv=s["max_kv"])
    return s["back"]


# -- what a pass cannot do without ------------------------------------------------------------------------------------

def work(case):
    c = case
    new, keys = lengths(c)
    M, H, KVH, D, e = sum(new), c["H"], c["KVH"], c["D"], SIZE[c["dtype"]]
    index = 8 * c["B"] + 4 * sum(-(-L // c["page"]) for L in keys)  # lengths and page numbers
    bytes_, flops = float(index), 0.0
    if c["op"] != "attn":
        bytes_ += M * (H + 2 * KVH) * D * SIZE[c["x"]] + M * 2 * KVH * D * e + 8 * c["rot"] // 2
        flops += M * (H + KVH) * (4.0 * c["norm"] * D + 3.0 * c["rot"])
    if c["op"] == "rope":  # only the pages that take new rows are looked up
        bytes_ += M * H * D * e - 4 * sum((L - n) // c["page"] for n, L in zip(new, keys))
    elif c["op"] == "attn":
        bytes_ += 2 * M * H * D * e + 2 * sum(keys) * KVH * D * e
    else:  # the new queries, keys and values stay on the chip at best
        bytes_ += M * H * D * e + 2 * (sum(keys) - M) * KVH * D * e
    if c["op"] != "rope":
        flops += 4.0 * H * D * _pairs(c)
    return dict(bytes=float(bytes_), flops=float(flops))


# -- the same in 64 bits ----------------------------------------------------------------------------------------------

def _exact_rope(c, d, new, keys):
    """Queries [M, H, D] and, for each sequence, its new keys and values [n, KVH, D], all in 64 bits."""
    H, KVH, D, rot = c["H"], c["KVH"], c["D"], c["rot"]
    x = d["qkv"].double().view(-1, H + 2 * KVH, D)
    place = torch.cat([torch.arange(L - n, L, device=DEV) for n, L in zip(new, keys)])
    freq, factor = _frequencies(rot, c["scaling"])
    turn = torch.polar(torch.full((), factor, device=DEV, dtype=torch.float64),
                       (d["pos"] if c["far"] else place).double().outer(freq))[:, None]
    first = torch.arange(0, rot, 2, device=DEV) if c["inter"] else torch.arange(rot // 2, device=DEV)
    second = first + (1 if c["inter"] else rot // 2)

    def side(v, w):
        if c["norm"]:
            v = v * torch.rsqrt(v.square().sum(-1, keepdim=True) / D + EPS) * w.double()
        z = torch.complex(v[..., first], v[..., second]) * turn
        v = v.clone()
        v[..., first], v[..., second] = z.real, z.imag
        return v

    k, v = side(x[:, H:H + KVH], d.get("wk")), x[:, H + KVH:]
    return side(x[:, :H], d.get("wq")), k, v


def _exact_cache(c, cache, rows, d, new, keys):
    """The cache in 64 bits with the new rows in their places."""
    out, m = cache.double(), 0
    for b, (n, L) in enumerate(zip(new, keys)):
        for p in range((L - n) // c["page"], -(-L // c["page"])):
            lo, hi = max(p * c["page"], L - n), min((p + 1) * c["page"], L)
            part = rows[m + lo - (L - n):m + hi - (L - n)].transpose(0, 1)
            out[d["table"][b, p].item(), :, lo - p * c["page"]:hi - p * c["page"]] = part
        m += n
    return out


def _exact_attention(c, q, kc, vc, d, new, keys):
    H, KVH, D, page = c["H"], c["KVH"], c["D"], c["page"]
    G, out, m = H // KVH, torch.zeros(sum(new), H, D, device=DEV, dtype=torch.float64), 0
    for b, (n, L) in enumerate(zip(new, keys)):
        pages = d["table"][b, :-(-L // page)].long()
        seen = L - n + 1 + torch.arange(n, device=DEV) if c["causal"] else torch.full((n,), L, device=DEV)
        for h in range(KVH):
            k = kc[pages, h].reshape(-1, D)[:L].double().t().contiguous()
            v = vc[pages, h].reshape(-1, D)[:L].double()
            for g in range(G):
                s = (q[m:m + n, h * G + g].double() / math.sqrt(D)) @ k
                s[torch.arange(L, device=DEV)[None] >= seen[:, None]] = -math.inf
                out[m:m + n, h * G + g] = torch.softmax(s, -1) @ v
        m += n
    return out.view(-1, H * D)


def exact(case, seed):
    c, d = case, _inputs(case, seed)
    new, keys = lengths(c)
    if c["op"] == "attn":
        return [_exact_attention(c, d["q"].view(-1, c["H"], c["D"]), d["kc"], d["vc"], d, new, keys)]
    q, k, v = _exact_rope(c, d, new, keys)
    kc, vc = _exact_cache(c, d["kc"], k, d, new, keys), _exact_cache(c, d["vc"], v, d, new, keys)
    if c["op"] == "rope":
        return [q.reshape(-1, c["H"] * c["D"]), kc, vc]
    t = TYPES[c["dtype"]]  # queries and the cache are held in their types
    return [_exact_attention(c, q.to(t), kc.to(t), vc.to(t), d, new, keys), kc, vc]
