"""Operators of MoE layers whose weights are 8-bit floating point (e4m3) with
one scale per 128 x 128 block, over activation rows in the same 8 bits with one
bf16 scale per 128 values (a scale needs range, not digits: the codes are
rounded against the scale as it is stored): the RMSNorm that takes the residual in and writes such
rows, the dense product, the two products grouped by expert over ragged
segments (gate/up with SwiGLU, down), and the weighted sum of the experts' rows.

`own` False: each operator in elementary torch operations, in 32 bits.  True:
the framework's calls (hip_backend over the C ABI) on the same tensors.

The shapes are the two MoE models this repository is built around (h 2048, 512
experts, top 10, ff 512; h 2048, 128 experts, top 8, ff 768) and the dense
projections beside them.
"""
import ctypes
import os
import sys

import torch

own = False

BLOCK = 128            # values that share a scale, of a row and of a weight block's sides
TOP = 448.0            # the largest e4m3 value
LEAST = 2.0 ** -126    # the smallest scale
EPS = 1e-6
STD = 0.02

NEXT = {"h": 2048, "E": 512, "K": 10, "ff": 512}
A3B = {"h": 2048, "E": 128, "K": 8, "ff": 768}


def listed():
    return [
        # the norm before a block: one token of a chat, and a long prompt
        {"kind": "norm", "name": "norm_token", "rows": 1, "n": 2048, "residual": True, "f32": True, "wtype": "f32"},
        {"kind": "norm", "name": "norm_prompt", "rows": 4096, "n": 2048, "residual": True, "f32": True, "wtype": "bf16"},
        # dense projections: one token, a batch of chats, a long prompt
        {"kind": "linear", "name": "linear_token", "tokens": 1, "in": 2048, "out": 4096, "scales": "f32", "y": "f32"},
        {"kind": "linear", "name": "linear_batch", "tokens": 24, "in": 4096, "out": 2048, "scales": "bf16", "y": "f32"},
        {"kind": "linear", "name": "linear_prompt", "tokens": 4001, "in": 2048, "out": 4096, "scales": "f32", "y": "bf16"},
        # the experts' gate and up products: one token, chats served at once
        # with a hot topic, a long prompt with popular experts
        dict(NEXT, kind="up", name="up_token", tokens=1, skew="none"),
        dict(NEXT, kind="up", name="up_batch", tokens=64, skew="hot"),
        dict(A3B, kind="up", name="up_prompt", tokens=4096, skew="zipf"),
        # and their down products: a small batch, a long prompt
        dict(A3B, kind="down", name="down_batch", tokens=24, skew="none", y="f32"),
        dict(NEXT, kind="down", name="down_prompt", tokens=4096, skew="none", y="bf16"),
        # the sum of each token's experts: a small batch, a long prompt
        {"kind": "mix", "name": "mix_batch", "tokens": 24, "h": 2048, "K": 8, "x": "f32", "residual": True},
        {"kind": "mix", "name": "mix_prompt", "tokens": 4096, "h": 2048, "K": 10, "x": "bf16", "residual": True},
    ]


def draw(rng):
    def size(lo, hi):
        return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))

    kind = rng.choice(["norm", "linear", "linear", "up", "up", "down", "down", "mix"])
    if kind == "norm":
        return {"kind": kind, "rows": size(1, 4096), "n": 16 * size(8, 256), "residual": rng.random() < 0.7,
                "f32": rng.random() < 0.5, "wtype": rng.choice(["f32", "bf16", "f16"])}
    if kind == "linear":
        n_in = rng.choice([512, 1024, 2048, 4096, 16 * size(8, 256)])
        out = rng.choice([256, 512, 2048, 4096, 2 * size(32, 2048)])
        return {"kind": kind, "tokens": size(1, 4096), "in": n_in, "out": out,
                "scales": rng.choice(["f32", "bf16", "f16"]), "y": rng.choice(["f32", "bf16"])}
    if kind == "mix":
        return {"kind": kind, "tokens": size(1, 4096), "h": 16 * size(8, 128), "K": rng.randint(1, 10),
                "x": rng.choice(["f32", "bf16"]), "residual": rng.random() < 0.5}
    c = dict(rng.choice([NEXT, A3B, {"h": 1024, "E": 64, "K": 6, "ff": 704},
                         {"h": 16 * size(16, 128), "E": size(4, 256), "K": rng.randint(1, 4), "ff": 16 * size(8, 48)}]),
             kind=kind, tokens=size(1, 4096), skew=rng.choice(["none", "hot", "zipf"]))
    if kind == "down":
        c["y"] = rng.choice(["f32", "bf16"])
    return c


# ------------------------------------------------------------------ inputs --
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def blocks(n):
    return -(-n // BLOCK)


def spread(s, rows, cols):
    """Block scales [..., rows / 128, cols / 128] as one value per element."""
    return s.repeat_interleave(BLOCK, -2)[..., :rows, :].repeat_interleave(BLOCK, -1)[..., :cols]


def spread_row(s, cols):
    return s.repeat_interleave(BLOCK, -1)[..., :cols]


def quantize(y):
    """Rows in 8 bits: (codes, scales), a scale being the largest magnitude of
    its 128 values over 448, rounded to bf16."""
    rows, n = y.shape
    p = torch.nn.functional.pad(y, (0, blocks(n) * BLOCK - n)).view(rows, blocks(n), BLOCK)
    s = (p.abs().amax(2) / TOP).clamp(min=LEAST).to(torch.bfloat16)
    return (y / spread_row(s.float(), n)).to(torch.float8_e4m3fn), s


def weights(gen, experts, out, n_in, stype):
    """N(0, 0.02) matrices in e4m3 with a scale per 128 x 128 block, the
    blocks' sizes spread as those of trained layers are."""
    bo, bi = blocks(out), blocks(n_in)
    codes = torch.empty(experts, out, n_in, dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty(experts, bo, bi, dtype=TYPES[stype], device="cuda")
    step = max(1, (1 << 28) // (out * n_in))
    for e in range(0, experts, step):
        n = min(step, experts - e)
        level = STD * torch.exp(0.3 * torch.randn(n, bo, bi, generator=gen, device="cuda"))
        w = torch.randn(n, out, n_in, generator=gen, device="cuda") * spread(level, out, n_in)
        p = torch.nn.functional.pad(w, (0, bi * BLOCK - n_in, 0, bo * BLOCK - out))
        top = p.view(n, bo, BLOCK, bi, BLOCK).abs().amax((2, 4))
        s = (top / TOP * 1.01).to(TYPES[stype])
        scales[e:e + n] = s
        codes[e:e + n] = (w / spread(s.float(), out, n_in)).to(torch.float8_e4m3fn)
    return codes, scales


def activations(gen, rows, n):
    """Rows of a residual stream: N(0, 1) with channels of unlike size."""
    return torch.randn(rows, n, generator=gen, device="cuda") * torch.exp(0.5 * torch.randn(n, generator=gen, device="cuda"))


def segments(gen, c):
    """Expert segments of a routing: offsets [E + 1], perm [P] (pair t * K + k
    of every position, an expert's pairs in order), and what the plain form
    needs to pad them: the experts in use and the longest segment."""
    T, E, K = c["tokens"], c["E"], c["K"]
    logits = torch.randn(T, E, generator=gen, device="cuda")
    if c["skew"] == "zipf":
        logits -= 1.1 * torch.log(torch.randperm(E, generator=gen, device="cuda").float() + 1)
    elif c["skew"] == "hot":
        hot = torch.randperm(E, generator=gen, device="cuda")[:16]
        logits[:, hot] += 8.0 * (torch.rand(T, 1, generator=gen, device="cuda") < 0.2)
    ids = logits.topk(K, 1).indices.reshape(-1)
    counts = torch.bincount(ids, minlength=E)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    return {"offsets": offsets.int(), "perm": torch.argsort(ids, stable=True).int(),
            "used": counts.nonzero().flatten(), "longest": int(counts.max())}


class State(dict):
    """A case's tensors, and what the framework's calls on them are issued with."""

    bound = None

    def __del__(self):
        if self.bound is not None:
            self.bound.drop()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000003 * seed + 17 * case.get("tokens", case.get("rows", 0)))
    s = State(case)
    kind = case["kind"]
    if kind == "norm":
        rows, n = case["rows"], case["n"]
        s["x"] = activations(gen, rows, n)
        s["r"] = activations(gen, rows, n) * 0.5 if case["residual"] else None
        s["w"] = (1.0 + 0.2 * torch.randn(n, generator=gen, device="cuda")).to(TYPES[case["wtype"]])
    elif kind == "linear":
        s["x8"], s["xs"] = quantize(activations(gen, case["tokens"], case["in"]))
        s["w8"], s["ws"] = (t[0] for t in weights(gen, 1, case["out"], case["in"], case["scales"]))
    elif kind == "mix":
        s["x"] = torch.randn(case["tokens"] * case["K"], case["h"], generator=gen, device="cuda").to(TYPES[case["x"]])
        s["w"] = torch.softmax(torch.randn(case["tokens"], case["K"], generator=gen, device="cuda"), 1)
        s["r"] = activations(gen, case["tokens"], case["h"]) if case["residual"] else None
    else:
        s.update(segments(gen, case))
        h, E, ff = case["h"], case["E"], case["ff"]
        if kind == "up":
            s["x8"], s["xs"] = quantize(activations(gen, case["tokens"], h))
            s["g8"], s["gs"] = weights(gen, E, ff, h, "f32")
            s["u8"], s["us"] = weights(gen, E, ff, h, "f32")
        else:
            a = torch.randn(2, case["tokens"] * case["K"], ff, generator=gen, device="cuda")
            s["x8"], s["xs"] = quantize(torch.sigmoid(a[0]) * a[0] * a[1])
            s["w8"], s["ws"] = weights(gen, E, h, ff, "f32")
    return s


# ---------------------------------------------------------- the plain forms --
def plain_norm(s):
    x = s["x"] if s["r"] is None else s["x"] + s["r"]
    y = x / torch.sqrt((x * x).mean(1, keepdim=True) + EPS) * s["w"].float()
    codes, scales = quantize(y)
    out = {"codes": codes, "scales": scales}
    if s["r"] is not None:
        out["sum"] = x
    if s["f32"]:
        out["y"] = y
    return out


def plain_linear(s):
    w = s["w8"].float() * spread(s["ws"].float(), s["out"], s["in"])
    x = s["x8"].float() * spread_row(s["xs"].float(), s["in"])
    return (x @ w.T).to(TYPES[s["y"]])


def padded(s):
    """Positions [used experts, longest segment] (past a segment's end: the
    last position) and, of every position, its expert's place and its row."""
    P = s["perm"].numel()
    off = s["offsets"].long()
    at = off[s["used"]][:, None] + torch.arange(s["longest"], device="cuda")
    p = torch.arange(P, device="cuda")
    e = torch.searchsorted(off[1:], p, right=True)
    place = torch.zeros(s["E"], dtype=torch.long, device="cuda")
    place[s["used"]] = torch.arange(s["used"].numel(), device="cuda")
    return at.clamp(max=P - 1), place[e], p - off[e]


def of_experts(s, codes, scales):
    c = codes[s["used"]]
    return c.float() * spread(scales[s["used"]].float(), c.shape[1], c.shape[2])


def plain_up(s):
    at, place, row = padded(s)
    x = s["x8"].float() * spread_row(s["xs"].float(), s["h"])
    x = x[s["perm"].long()[at] // s["K"]]
    g = torch.bmm(x, of_experts(s, s["g8"], s["gs"]).transpose(1, 2).contiguous())
    u = torch.bmm(x, of_experts(s, s["u8"], s["us"]).transpose(1, 2).contiguous())
    codes, scales = quantize((g / (1.0 + torch.exp(-g)) * u)[place, row])
    return {"codes": codes, "scales": scales}


def plain_down(s):
    at, place, row = padded(s)
    x = (s["x8"].float() * spread_row(s["xs"].float(), s["ff"]))[at]
    y = torch.bmm(x, of_experts(s, s["w8"], s["ws"]).transpose(1, 2).contiguous())
    out = torch.empty(s["perm"].numel(), s["h"], dtype=TYPES[s["y"]], device="cuda")
    out[s["perm"].long()] = y[place, row].to(out.dtype)
    return out


def plain_mix(s):
    x = s["x"].float().view(s["tokens"], s["K"], s["h"])
    y = (x * s["w"][..., None]).sum(1)
    return y if s["r"] is None else y + s["r"]


# ------------------------------------------------------ the framework's calls --
OPEN = {}


def batch():
    """The one open batch that passes are issued in, as a serving loop's."""
    if not OPEN:
        pkg = os.path.join(os.getcwd(), "llama-rs-metal_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import hip_backend

        OPEN["gpu"] = hip_backend.Gpu()
        OPEN["batch"] = hip_backend.Batch(OPEN["gpu"])
    return OPEN["gpu"], OPEN["batch"]


class Bound:
    """A state's tensors adopted in place (moe_register) under the framework's
    types, and its output buffers."""

    def __init__(self, s):
        self.gpu, self.batch = batch()
        import hip_backend as hb

        self.hb, self.kept = hb, []
        kind, f32 = s["kind"], torch.float32
        if kind == "norm":
            rows, n = s["rows"], s["n"]
            self.codes, self.scales, self.q = self.rows_out(rows, n)
            self.out = {"codes": self.codes, "scales": self.scales}
            self.x, self.r = self.buffer(s["x"]), self.maybe(s["r"])
            self.w = self.weight(s["w"], None, [n], s["wtype"])
            self.sum = self.y = None
            if s["r"] is not None:
                self.out["sum"] = torch.empty(rows, n, device="cuda")
                self.sum = self.buffer(self.out["sum"])
            if s["f32"]:
                self.out["y"] = torch.empty(rows, n, device="cuda")
                self.y = self.buffer(self.out["y"])
        elif kind == "linear":
            self.x = self.rows(s["x8"], s["xs"])
            self.w = self.weight(s["w8"], s["ws"], [s["in"], s["out"]], s["scales"])
            self.out = torch.empty(s["tokens"], s["out"], dtype=TYPES[s["y"]], device="cuda")
            self.y, self.ytype = self.buffer(self.out), hb.F32 if s["y"] == "f32" else hb.BF16
        elif kind == "mix":
            self.x, self.xtype = self.buffer(s["x"]), hb.F32 if s["x"].dtype == f32 else hb.BF16
            self.w, self.r = self.buffer(s["w"]), self.maybe(s["r"])
            self.out = torch.empty(s["tokens"], s["h"], dtype=f32, device="cuda")
            self.y = self.buffer(self.out)
        else:
            h, E, ff = s["h"], s["E"], s["ff"]
            P = s["perm"].numel()
            self.x = self.rows(s["x8"], s["xs"])
            self.offsets, self.perm = self.buffer(s["offsets"]), self.buffer(s["perm"])
            if kind == "up":
                self.gate = self.weight(s["g8"], s["gs"], [h, ff, E], "f32")
                self.up = self.weight(s["u8"], s["us"], [h, ff, E], "f32")
                self.codes, self.scales, self.q = self.rows_out(P, ff)
                self.out = {"codes": self.codes, "scales": self.scales}
            else:
                self.w = self.weight(s["w8"], s["ws"], [ff, h, E], "f32")
                self.out = torch.empty(P, h, dtype=TYPES[s["y"]], device="cuda")
                self.y, self.ytype = self.buffer(self.out), hb.F32 if s["y"] == "f32" else hb.BF16
        # the engine's stream does not wait for torch's, which makes the inputs
        torch.cuda.current_stream().synchronize()

    def adopt(self, t):
        lib = self.hb.load_library()
        if lib.moe_register(self.gpu._h, ctypes.c_void_p(t.data_ptr()), t.numel() * t.element_size()) != 0:
            raise RuntimeError(lib.moe_last_error(self.gpu._h).decode())
        self.kept.append(t)

    def buffer(self, t):
        from hip_backend.api import MoeBufferC

        self.adopt(t)
        return self.hb.Buffer(self.gpu, MoeBufferC(t.data_ptr(), t.numel() * t.element_size() // 4), t.data_ptr())

    def maybe(self, t):
        return None if t is None else self.buffer(t)

    def region(self, t):
        from hip_backend.api import MoeRegionC

        self.adopt(t)
        return MoeRegionC(t.data_ptr(), t.numel() * t.element_size())

    def rows(self, codes, scales):
        return self.hb.Rows8(self.region(codes), self.region(scales), codes.shape[0], codes.shape[1])

    def rows_out(self, rows, n):
        codes = torch.empty(rows, n, dtype=torch.float8_e4m3fn, device="cuda")
        scales = torch.empty(rows, blocks(n), dtype=torch.bfloat16, device="cuda")
        return codes, scales, self.rows(codes, scales)

    def weight(self, t, scales, dims, kind):
        from hip_backend.api import MoeWeightC

        hb, c = self.hb, MoeWeightC()
        kind = {"f32": hb.F32, "f16": hb.F16, "bf16": hb.BF16}[kind]
        c.data, c.ndims = self.region(t), len(dims)
        c.dims[:len(dims)] = dims
        if scales is None:
            c.dtype = kind
        else:
            c.scales = self.region(scales)
            c.dtype, c.group_size, c.scale_type = hb.E4M3, BLOCK, kind
        return hb.Weight(c, [c.data], dims, 0)

    def drop(self):
        """Takes the tensors back when no pass is left that reads or writes them."""
        try:
            torch.cuda.synchronize()
            lib = self.hb.load_library()
            self.kept = [t for t in self.kept if lib.moe_unregister(self.gpu._h, ctypes.c_void_p(t.data_ptr())) != 0]
        except (TypeError, AttributeError):
            pass  # the interpreter is ending: its modules and the engine are gone


def own_run(s):
    """The calls go to the engine's own stream: who reads their outputs with torch
    waits for the device first."""
    if s.bound is None:
        s.bound = Bound(s)
    b, o = s.bound.batch, s.bound
    kind = s["kind"]
    if kind == "norm":
        b.norm_q8(o.x, o.r, o.w, o.sum, o.y, o.q, EPS)
    elif kind == "linear":
        b.matmul_q8(o.w, o.x, o.y, o.ytype)
    elif kind == "mix":
        b.mix_tokens(o.x, o.w, o.r, o.y, s["tokens"], o.xtype)
    elif kind == "up":
        b.expert_swiglu_q8(o.gate, o.up, o.x, o.offsets, o.perm, s["K"], o.q)
    else:
        b.expert_matmul_q8(o.w, o.x, o.offsets, o.perm, o.y, o.ytype)
    return o.out


def run(state):
    if own:
        return own_run(state)
    return {"norm": plain_norm, "linear": plain_linear, "up": plain_up, "down": plain_down,
            "mix": plain_mix}[state["kind"]](state)


# ------------------------------------------------------------- work, exact --
def used_experts(c):
    """Experts that a routing of this skew is expected to use."""
    E, K, T = c["E"], c["K"], c["tokens"]
    if c["skew"] == "zipf":
        p = [(e + 1) ** -1.1 for e in range(E)]
        return sum(1.0 - (1.0 - min(1.0, K * q / sum(p))) ** T for q in p)
    if c["skew"] == "hot" and T > 4 and E > 16:
        return min(E, 16 + (E - 16) * (1.0 - (1.0 - K / E) ** (0.8 * T)))
    return E * (1.0 - (1.0 - K / E) ** T)


def work(case):
    def rows8(rows, n):
        return rows * (n + 2 * blocks(n))

    kind = case["kind"]
    if kind == "norm":
        rows, n = case["rows"], case["n"]
        by = rows * n * 4 * (1 + 2 * case["residual"] + case["f32"]) + rows8(rows, n) + n * TYPES[case["wtype"]].itemsize
        return {"bytes": by, "flops": 8 * rows * n}
    if kind == "linear":
        T, i, o = case["tokens"], case["in"], case["out"]
        by = rows8(T, i) + o * i + blocks(o) * blocks(i) * TYPES[case["scales"]].itemsize
        return {"bytes": by + T * o * TYPES[case["y"]].itemsize, "flops": 2 * T * i * o}
    T, K, h = case["tokens"], case["K"], case["h"]
    if kind == "mix":
        return {"bytes": T * K * (h * TYPES[case["x"]].itemsize + 4) + 4 * T * h * (1 + case["residual"]),
                "flops": 2 * T * K * h}
    ff = case["ff"]
    one = h * ff + 4 * blocks(h) * blocks(ff)
    if kind == "up":
        return {"bytes": int(2 * used_experts(case) * one) + rows8(T, h) + rows8(T * K, ff) + 4 * T * K,
                "flops": 4 * T * K * h * ff}
    return {"bytes": int(used_experts(case) * one) + rows8(T * K, ff) + T * K * (h * TYPES[case["y"]].itemsize + 4),
            "flops": 2 * T * K * h * ff}


def exact(case, seed):
    """The outputs in 64 bits from the definition, codes and scales before they
    are rounded."""
    s = prepare(case, seed)
    f64 = torch.float64

    def value(codes, scales, sides):
        v = codes.to(f64)
        up = scales.to(f64)
        for d in range(sides):
            up = torch.repeat_interleave(up, BLOCK, dim=up.dim() - 1 - d)
        return v * (up[:v.shape[0], :v.shape[1]] if sides == 2 else up[:, :v.shape[1]])

    def coded(y):
        n = y.shape[1]
        scale = torch.stack([g.abs().max(1).values for g in y.split(BLOCK, 1)], 1) / TOP
        return {"codes": torch.cat([g / scale[:, i:i + 1] for i, g in enumerate(y.split(BLOCK, 1))], 1)[:, :n],
                "scales": scale}

    kind = case["kind"]
    if kind == "norm":
        x = s["x"].to(f64)
        if s["r"] is not None:
            x = x + s["r"].to(f64)
        y = x * s["w"].to(f64) / (x.pow(2).sum(1, keepdim=True) / case["n"] + EPS).sqrt()
        out = coded(y)
        if s["r"] is not None:
            out["sum"] = x
        if case["f32"]:
            out["y"] = y
        return out
    if kind == "linear":
        return value(s["x8"], s["xs"], 1) @ value(s["w8"], s["ws"], 2).T
    if kind == "mix":
        y = torch.zeros(case["tokens"], case["h"], dtype=f64, device="cuda")
        for k in range(case["K"]):
            y += s["x"][k::case["K"]].to(f64) * s["w"][:, k:k + 1].to(f64)
        return y if s["r"] is None else y + s["r"].to(f64)
    x = value(s["x8"], s["xs"], 1)
    off, perm = s["offsets"].tolist(), s["perm"].long()
    y = torch.zeros(perm.numel(), case["ff"] if kind == "up" else case["h"], dtype=f64, device="cuda")
    for e in range(case["E"]):
        lo, hi = off[e], off[e + 1]
        if lo == hi:
            continue
        if kind == "up":
            a = x[torch.div(perm[lo:hi], case["K"], rounding_mode="floor")]
            g = a @ value(s["g8"][e], s["gs"][e], 2).T
            y[lo:hi] = g * torch.sigmoid(g) * (a @ value(s["u8"][e], s["us"][e], 2).T)
        else:
            y[perm[lo:hi]] = x[lo:hi] @ value(s["w8"][e], s["ws"][e], 2).T
    return coded(y) if kind == "up" else y
