"""The feed-forward operators on real work: the gated linear block (forward and training
step) and the microscaled 4-bit (MXFP4) quantisation, product and gated block.

`run` with `own` false is each operator's plain form: elementary torch operations in 32
bits, rounded once at the end.  With `own` true it makes the calls that a user makes of
`xvram_b200.torch_bridge`.

  gated block   h = act(x Wg^T + bg) * (x Wu^T + bu), x (m, d), Wg and Wu (h, d)
  MXFP4         blocks of 32 along a row share a scale 2^(s - 127),
                s = clamp(floor(log2 max|x|) - 2, -127, 127) + 127; the elements are E2M1
                (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives), nearest, ties to even,
                saturating.  Two codes to a byte, the even element in the low half; scales in
                tiles of 128 rows x 4 blocks: byte (r % 32) * 16 + (r / 32 % 4) * 4 + b % 4 of
                tile (r / 128, b / 4).  Padding codes are 0 and padding scales 127.
  linear        y = Q(x) W^T + bias (then ReLU), with Q(x) the MXFP4 values of x
"""
import math

import torch

own = False

BLOCK = 32
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ACTS = ("silu", "gelu", "gelu_tanh", "relu", "sigmoid")


def listed():
    return [
        # One token of a small model: launch latency next to 8 MB of weights.
        {"name": "gated_token_bf16", "op": "gated", "m": 1, "d": 1024, "h": 2048, "type": "bf16", "act": "silu", "bias": False},
        # A decode step of a small batch: bound by reading the two weights.
        {"name": "gated_decode_fp16", "op": "gated", "m": 24, "d": 4096, "h": 8192, "type": "fp16", "act": "gelu_tanh", "bias": False},
        # A prompt or an evaluation batch.
        {"name": "gated_batch_bf16", "op": "gated", "m": 2048, "d": 4096, "h": 8192, "type": "bf16", "act": "silu", "bias": False},
        # A few rows of odd sizes in the framework's own type, with biases.
        {"name": "gated_ragged_fp32", "op": "gated", "m": 5, "d": 2047, "h": 4099, "type": "fp32", "act": "sigmoid", "bias": True},
        # A training step: forward, and the gradients of the input and both weights.
        {"name": "train_bf16", "op": "train", "m": 8192, "d": 4096, "h": 8192, "type": "bf16", "act": "silu", "bias": False},
        # A training step of odd sizes with biases: no dimension is a whole number of tiles.
        {"name": "train_ragged_fp16", "op": "train", "m": 1021, "d": 1001, "h": 2730, "type": "fp16", "act": "gelu", "bias": True},
        # A large weight brought to 4 bits, and read back.
        {"name": "quantise_bf16", "op": "quantise", "m": 4096, "d": 16384, "type": "bf16"},
        # Few rows that end inside a block.
        {"name": "quantise_ragged_fp32", "op": "quantise", "m": 333, "d": 1001, "type": "fp32"},
        # One token through a wide 4-bit layer.
        {"name": "mx_linear_token_bf16", "op": "mx_linear", "m": 1, "d": 4096, "h": 16384, "type": "bf16", "bias": False, "relu": False},
        # The streamed MLP's layer: 16384 features, batch 512, bias and ReLU.
        {"name": "mx_linear_layer_bf16", "op": "mx_linear", "m": 512, "d": 16384, "h": 16384, "type": "bf16", "bias": True, "relu": True},
        # A decode step of the gated block with 4-bit weights.
        {"name": "mx_gated_decode_bf16", "op": "mx_gated", "m": 16, "d": 4096, "h": 8192, "type": "bf16", "act": "silu", "bias": False},
        # A long prompt through the gated block with 4-bit weights.
        {"name": "mx_gated_prompt_fp16", "op": "mx_gated", "m": 4096, "d": 4096, "h": 8192, "type": "fp16", "act": "gelu_tanh", "bias": True},
    ]


def _size(rng, low, high):
    """Spread over the logarithm; two in five are odd sizes, the others whole multiples of 64
    where they are large enough."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.4:
        return max(low, min(high, v | 1 if v < high else v - 1))
    return max(low, min(high, v // 64 * 64 if v >= 128 else v))


def draw(rng):
    op = rng.choice(["gated", "gated", "train", "quantise", "mx_linear", "mx_gated"])
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "quantise":
        return {"op": op, "m": _size(rng, 1, 8192), "d": _size(rng, 32, 8192), "type": kind}
    # 32-bit products run on the FP32 units, so their largest sizes are smaller; a 4-bit product's
    # activations are of 16 bits.
    if op.startswith("mx_") and kind == "fp32":
        kind = "bf16"
    most = 2.0 ** 38 if kind != "fp32" else 2.0 ** 32
    while True:
        m, d, h = _size(rng, 1, 8192), _size(rng, 64, 16384), _size(rng, 64, 16384)
        if m * d * h <= most:
            break
    case = {"op": op, "m": m, "d": d, "h": h, "type": kind, "bias": rng.random() < 0.5}
    if op == "mx_linear":
        case["relu"] = rng.random() < 0.5
    else:
        case["act"] = rng.choice(ACTS)
    return case


# ---------------------------------------------------------------- inputs
def _powers(e):
    """2^e in float32 for whole e in [-126, 127]."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _mx(x):
    """(signed E2M1 values, block exponents) of x's rows, in 32 bits, the last block padded with
    zeros."""
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    if blocks * BLOCK != cols:
        x = torch.cat([x, x.new_zeros(rows, blocks * BLOCK - cols)], 1)
    x = x.view(rows, blocks, BLOCK)
    top = x.abs().amax(2)
    e = torch.where(top > 0, (torch.frexp(top)[1] - 3).clamp(min=-126), torch.full_like(top, -126, dtype=torch.int32))
    a = (x * _powers(-e)[..., None])
    size = a.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    q = torch.clamp(torch.round(size / step) * step, max=6.0)
    return torch.where(a < 0, -q, q), e


def _mx_values(x):
    q, e = _mx(x)
    return (q * _powers(e)[..., None]).flatten(1)[:, :x.shape[1]].contiguous()


def _mx_pack(x):
    """(codes, scales) of x in the stored form."""
    q, e = _mx(x)
    rows, blocks = e.shape
    code = torch.tensor([0, 1, 2, 3, 4, 0, 5, 0, 6, 0, 0, 0, 7], dtype=torch.uint8, device=x.device)[(q.abs() * 2).long()]
    code = (code + 8 * (q < 0).to(torch.uint8)).flatten(1)
    codes = (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous()
    tr, tb = -(-rows // 128), -(-blocks // 4)
    s = torch.full((tr * 128, tb * 4), 127, dtype=torch.uint8, device=x.device)
    s[:rows, :blocks] = (e + 127).to(torch.uint8)
    scales = s.view(tr, 4, 32, tb, 4).permute(0, 3, 2, 1, 4).contiguous().view(tr, tb, 512)
    return codes, scales


def _mx_unpack(codes, scales, rows, cols):
    """The values that stored codes and scales stand for, in 32 bits."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float32, device=codes.device)
    q = torch.stack([table[(codes & 15).long()], table[(codes >> 4).long()]], 2).flatten(1)
    tr, tb = scales.shape[:2]
    s = scales.view(tr, tb, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(tr * 128, tb * 4)[:rows, :q.shape[1] // BLOCK]
    return (q.view(rows, -1, BLOCK) * _powers(s.to(torch.int32) - 127)[..., None]).flatten(1)[:, :cols]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, op, m, d = TYPES[case["type"]], case["op"], case["m"], case["d"]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device="cuda") * scale

    s = {"case": dict(case)}
    if op == "quantise":
        # Weights: features of different sizes, a few outliers, and some blocks of zeros.
        w = normal(m, d) * torch.exp(normal(m, 1))
        w = w * torch.where(torch.rand((m, d), generator=g, device="cuda") < 0.001, 30.0, 1.0)
        keep = torch.rand((m, -(-d // BLOCK)), generator=g, device="cuda") > 0.002
        s["x"] = (w * keep.repeat_interleave(BLOCK, 1)[:, :d]).to(t)
        return s
    h = case["h"]
    s["x"] = normal(m, d).to(t)
    names = ("w",) if op == "mx_linear" else ("w_gate", "w_up")
    for n in names:
        w = normal(h, d, scale=d ** -0.5)
        s[n] = _mx_pack(w) if op.startswith("mx_") else w.to(t)
        s[n.replace("w", "b", 1)] = normal(h, scale=0.5).to(t) if case["bias"] else None
    if op == "train":
        s["dh"] = normal(m, h).to(t)
        for n in ("x", "w_gate", "w_up", "b_gate", "b_up"):
            if s[n] is not None:
                s[n].requires_grad_()
    return s


# ---------------------------------------------------------------- plain forms
def _act(v, act):
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-v))
    if act == "relu":
        return torch.clamp(v, min=0)
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))


def _slope(v, act):
    """act'(v)."""
    if act == "silu":
        q = 1 / (1 + torch.exp(-v))
        return q * (1 + v * (1 - q))
    if act == "sigmoid":
        q = 1 / (1 + torch.exp(-v))
        return q * (1 - q)
    if act == "relu":
        return (v > 0).to(v.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(v * math.sqrt(0.5))) + v * torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    q = torch.tanh(c * (v + 0.044715 * v * v * v))
    return 0.5 * (1 + q) + 0.5 * v * (1 - q * q) * c * (1 + 3 * 0.044715 * v * v)


def _project(x, w, b):
    y = x @ w.t()
    return y if b is None else y + b.float()


def _plain(s):
    c = s["case"]
    t, op, m, d = TYPES[c["type"]], c["op"], c["m"], c["d"]
    if op == "quantise":
        return {"values": _mx_values(s["x"].float())}
    if op == "mx_linear":
        y = _project(_mx_values(s["x"].float()), _mx_unpack(*s["w"], c["h"], d), s["b"])
        return {"y": (torch.clamp(y, min=0) if c["relu"] else y).to(t)}
    if op == "mx_gated":
        x = _mx_values(s["x"].float())
        g = _project(x, _mx_unpack(*s["w_gate"], c["h"], d), s["b_gate"])
        u = _project(x, _mx_unpack(*s["w_up"], c["h"], d), s["b_up"])
        return {"h": (_act(g, c["act"]) * u).to(t)}
    x, wg, wu = (s[n].detach().float() for n in ("x", "w_gate", "w_up"))
    bg, bu = (None if s[n] is None else s[n].detach() for n in ("b_gate", "b_up"))
    g, u = _project(x, wg, bg), _project(x, wu, bu)
    a = _act(g, c["act"])
    out = {"h": (a * u).to(t)}
    if op == "train":
        dh = s["dh"].float()
        dg, du = dh * u * _slope(g, c["act"]), dh * a
        out |= {"dx": (dg @ wg + du @ wu).to(t), "dw_gate": (dg.t() @ x).to(t), "dw_up": (du.t() @ x).to(t)}
        if c["bias"]:
            out |= {"db_gate": dg.sum(0).to(t), "db_up": du.sum(0).to(t)}
    return out


# ---------------------------------------------------------------- the framework's calls
def _own(s):
    from xvram_b200 import torch_bridge as tb
    c = s["case"]
    op = c["op"]
    if op == "quantise":
        return {"values": tb.dequantize_mxfp4(tb.quantize_mxfp4(s["x"]))}
    if op == "mx_linear":
        w = tb.Mxfp4Matrix(*s["w"], (c["h"], c["d"]))
        return {"y": tb.linear_mxfp4(s["x"], w, s["b"], relu=c["relu"])}
    if op == "mx_gated":
        w = [tb.Mxfp4Matrix(*s[n], (c["h"], c["d"])) for n in ("w_gate", "w_up")]
        return {"h": tb.gated_linear_mxfp4(s["x"], *w, s["b_gate"], s["b_up"], activation=c["act"])}
    if op == "gated":
        return {"h": tb.gated_linear(s["x"], s["w_gate"], s["w_up"], s["b_gate"], s["b_up"], activation=c["act"])}
    leaves = ["x", "w_gate", "w_up"] + (["b_gate", "b_up"] if c["bias"] else [])
    h = tb.gated_linear(s["x"], s["w_gate"], s["w_up"], s["b_gate"], s["b_up"], activation=c["act"])
    grads = torch.autograd.grad(h, [s[n] for n in leaves], s["dh"])
    return {"h": h.detach()} | {"d" + n: v for n, v in zip(leaves, grads)}


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------- work and exact values
def work(case):
    m, d, op = case["m"], case["d"], case["op"]
    size = TYPES[case["type"]].itemsize
    if op == "quantise":
        # The source in, codes and scales out and in again, and the values out.
        stored = m * -(-d // BLOCK) * 17
        return {"bytes": m * d * (size + 4) + 2 * stored, "flops": 0}
    h, n = case["h"], 1 if op == "mx_linear" else 2
    weight = h * -(-d // BLOCK) * 17 if op.startswith("mx_") else h * d * size
    bias = n * h * size if case["bias"] else 0
    nbytes, flops = m * d * size + n * weight + bias + m * h * size, 2 * n * m * d * h
    if op == "train":
        nbytes += m * h * size + m * d * size + n * weight + bias
        flops *= 3
    return {"bytes": nbytes, "flops": flops}


def _nearest(x):
    """MXFP4 values of x in 64 bits: each element's nearest E2M1 value by comparison with all
    of them, the even code where two are as near."""
    x = x.double()
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    x = torch.cat([x, x.new_zeros(rows, blocks * BLOCK - cols)], 1).view(rows, blocks, BLOCK)
    top = x.abs().amax(2, keepdim=True)
    # floor(log2) from the exponent's bits: a logarithm's last place would decide powers of two.
    e = torch.clamp((top.view(torch.int64) >> 52) - 1023 - 2, min=-127)
    scale = ((e + 1023) << 52).view(torch.float64)
    a = x.abs() / scale
    value = torch.zeros_like(a)
    for i in range(1, 8):  # up to value i from the midpoint on, where the midpoint goes to an even code
        middle = (E2M1[i] + E2M1[i - 1]) / 2
        value = torch.where(a >= middle if i % 2 == 0 else a > middle, E2M1[i], value)
    return (torch.where(x < 0, -value, value) * scale).flatten(1)[:, :cols]


def _stored(codes, scales, rows, cols):
    """The values of stored codes and scales in 64 bits, by each element's own address."""
    r = torch.arange(rows, device=codes.device)[:, None]
    k = torch.arange(cols, device=codes.device)[None, :]
    code = (codes[r, k // 2].int() >> (4 * (k % 2))) & 15
    b = k // BLOCK
    s = scales[r // 128, b // 4, (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4].double()
    e, f = ((code >> 1) & 3).double(), (code & 1).double()
    size = torch.where(e > 0, torch.exp2(e - 1) * (1 + f / 2), f / 2)
    return torch.where(code > 7, -size, size) * torch.exp2(s - 127)


def exact(case, seed):
    s = prepare(case, seed)
    op, m, d = case["op"], case["m"], case["d"]
    if op == "quantise":
        return {"values": _nearest(s["x"])}
    acts = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu, "sigmoid": torch.sigmoid,
            "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}

    def bias(n):
        return 0.0 if s[n] is None else s[n].double()

    if op.startswith("mx_"):
        x = _nearest(s["x"])
        if op == "mx_linear":
            y = x @ _stored(*s["w"], case["h"], d).t() + bias("b")
            return {"y": torch.relu(y) if case["relu"] else y}
        g = x @ _stored(*s["w_gate"], case["h"], d).t() + bias("b_gate")
        return {"h": acts[case["act"]](g) * (x @ _stored(*s["w_up"], case["h"], d).t() + bias("b_up"))}
    leaves = {n: s[n].detach().double().requires_grad_(op == "train") for n in ("x", "w_gate", "w_up", "b_gate", "b_up") if s[n] is not None}
    g = torch.nn.functional.linear(leaves["x"], leaves["w_gate"], leaves.get("b_gate"))
    h = acts[case["act"]](g) * torch.nn.functional.linear(leaves["x"], leaves["w_up"], leaves.get("b_up"))
    if op == "gated":
        return {"h": h}
    grads = torch.autograd.grad(h, list(leaves.values()), s["dh"].double())
    return {"h": h.detach()} | {"d" + n: v for n, v in zip(leaves, grads)}
