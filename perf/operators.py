"""Cases, plain forms and exact values of the operators around the MoE layer:

  route    group-limited routing: router logits -> expert ids and weights
  linear   FP8 matrix product with 1x128 activation and 128x128 weight scales
  gate_up  the same product with gate/up columns, silu(gate) * up, re-quantised 1x128
  mlp      gate_up, then linear, plus a residual: a dense or shared expert

`own` selects the framework's kernels; otherwise elementary torch operations."""
import math

import torch

own = False

DEV = "cuda"
FP8 = torch.float8_e4m3fn
BLOCK = 128


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _route(name, M, E, groups, topk_group, k, scoring, bias, bf16=False, scale=2.5):
    return {"name": name, "op": "route", "M": M, "E": E, "groups": groups, "topk_group": topk_group, "k": k,
            "scoring": scoring, "bias": bias, "bf16": bf16, "scale": scale}


def _linear(name, M, N, K, quantized, f32=False, residual=False):
    return {"name": name, "op": "linear", "M": M, "N": N, "K": K, "quantized": quantized, "f32": f32,
            "residual": residual}


def _gate_up(name, M, H, I, quantized):
    return {"name": name, "op": "gate_up", "M": M, "H": H, "I": I, "quantized": quantized}


def _mlp(name, M, H, I, residual):
    return {"name": name, "op": "mlp", "M": M, "H": H, "I": I, "residual": residual}


def listed():
    return [
        # one decoded token through a 256-expert router with a balance bias: latency
        _route("route 1 token", 1, 256, 8, 4, 8, "sigmoid", True),
        # a prefill batch through the same router: bandwidth
        _route("route 8192 tokens", 8192, 256, 8, 4, 8, "sigmoid", True),
        # softmax router with bf16 logits, groups of 20 experts, an odd number of tokens
        _route("route softmax 1001 tokens", 1001, 160, 8, 3, 6, "softmax", False, bf16=True, scale=16.0),
        # one decoded token through a projection of the GLM layer's width
        _linear("linear 1 token", 1, 4096, 6144, False),
        # a decode batch through the shared expert's down-projection, added to the routed output
        _linear("linear 64 tokens", 64, 6144, 2048, True, residual=True),
        # odd sizes: a narrow projection whose rows end inside a scale block, f32 out
        _linear("linear 333 tokens", 333, 576, 7168, True, f32=True),
        # a prefill chunk through a square projection: tensor-core rate
        _linear("linear 8192 tokens", 8192, 6144, 6144, True),
        # a small decode batch through the shared expert's gate/up projection
        _gate_up("gate_up 16 tokens", 16, 6144, 2048, False),
        # a prefill chunk through it
        _gate_up("gate_up 4096 tokens", 4096, 6144, 2048, True),
        # one decoded token through the whole shared expert
        _mlp("mlp 1 token", 1, 6144, 2048, True),
        # a ragged mid-size batch through it, as in a chunked prefill
        _mlp("mlp 200 tokens", 200, 6144, 2048, True),
        # a prefill chunk through a wide dense feed-forward layer
        _mlp("mlp 2048 tokens", 2048, 7168, 18432, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _log128(rng, lo, hi):
    return BLOCK * _log(rng, lo // BLOCK, hi // BLOCK)


MOST_FLOPS = 1.5e12


def _tokens(rng, flops_per_token):
    return _log(rng, 1, max(1, min(8192, int(MOST_FLOPS / flops_per_token))))


def draw(rng):
    op = rng.choice(("route", "linear", "gate_up", "mlp"))
    if op == "route":
        groups = rng.choice((1, 2, 4, 8, 16))
        per = rng.randint(2, 512 // groups)
        topk_group = rng.randint(1, groups)
        k = rng.randint(1, min(16, topk_group * per))
        sigmoid = rng.random() < 0.6
        return {"op": op, "M": _log(rng, 1, 8192), "E": groups * per, "groups": groups, "topk_group": topk_group,
                "k": k, "scoring": "sigmoid" if sigmoid else "softmax", "bias": sigmoid and rng.random() < 0.7,
                "bf16": rng.random() < 0.4, "scale": rng.choice((1.0, 2.5))}
    if op == "linear":
        N, K = _log(rng, 1, 8192), _log128(rng, 128, 8192)
        return {"op": op, "M": _tokens(rng, 2 * N * K), "N": N, "K": K, "quantized": rng.random() < 0.5,
                "f32": rng.random() < 0.3, "residual": rng.random() < 0.4}
    H, I = _log128(rng, 256, 8192), _log128(rng, 128, 16384)
    if op == "gate_up":
        return {"op": op, "M": _tokens(rng, 4 * H * I), "H": H, "I": I, "quantized": rng.random() < 0.5}
    return {"op": op, "M": _tokens(rng, 6 * H * I), "H": H, "I": I, "residual": rng.random() < 0.5}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _f32_div(a, b):
    """IEEE division: torch multiplies by the reciprocal when b is a Python number."""
    return a / torch.full((), b, dtype=a.dtype, device=a.device)


def _quant_rows(x):
    """1x128 quantisation of (M, K): codes and f32 scales."""
    M, K = x.shape
    v = x.float().reshape(M, K // BLOCK, BLOCK)
    s = _f32_div(v.abs().amax(-1), 448.0).clamp_min(1e-12)
    q = (v / s.unsqueeze(-1)).clamp(-448.0, 448.0).to(FP8).reshape(M, K)
    return q, s


def _weight(g, N, K):
    """A weight (N, K) of a projection as a checkpoint holds it: e4m3 codes and one f32 scale per 128x128 block."""
    nb, kb = -(-N // BLOCK), K // BLOCK
    w = torch.randn(nb * BLOCK, K, generator=g, device=DEV, dtype=torch.bfloat16).mul_(K ** -0.5)
    v = w.view(nb, BLOCK, kb, BLOCK)
    s = _f32_div(v.abs().amax(dim=(1, 3)).float(), 448.0).clamp_min(1e-12)
    q = (v.float() / s[:, None, :, None]).clamp_(-448.0, 448.0).to(FP8).reshape(nb * BLOCK, K)
    return q[:N].contiguous(), s


def _hidden(g, M, K):
    """Activations of M tokens: unit normal, each token with a size of its own and a few large channels."""
    x = torch.randn(M, K, generator=g, device=DEV)
    x *= torch.exp(0.5 * torch.randn(M, 1, generator=g, device=DEV))
    x *= 1.0 + 20.0 * (torch.rand(1, K, generator=g, device=DEV) < 0.004)
    return x.to(torch.bfloat16)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    st = {"case": case}
    op = case["op"]
    if op == "route":
        x = 1.5 * torch.randn(case["M"], case["E"], generator=g, device=DEV)
        st["logits"] = x.to(torch.bfloat16) if case["bf16"] else x
        st["bias"] = 0.1 * torch.randn(case["E"], generator=g, device=DEV) if case["bias"] else None
        return st
    K = case["K"] if op == "linear" else case["H"]
    x, xs = _hidden(g, case["M"], K), None
    if case.get("quantized"):
        x, xs = _quant_rows(x)
    st["x"], st["xs"] = x, xs
    if op == "linear":
        st["w"], st["ws"] = _weight(g, case["N"], K)
    else:
        st["w13"], st["w13s"] = _weight(g, 2 * case["I"], K)
        if op == "mlp":
            st["w2"], st["w2s"] = _weight(g, K, case["I"])
    if case.get("residual"):
        n = case["N"] if op == "linear" else K
        st["residual"] = torch.randn(case["M"], n, generator=g, device=DEV).to(torch.bfloat16)
    return st


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _plain_route(st):
    c = st["case"]
    M, E, G = c["M"], c["E"], c["groups"]
    x = st["logits"].double()
    # scores in 64 bits: values next to the border decide which expert is taken
    if c["scoring"] == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-x))
    else:
        e = torch.exp(x - x.amax(1, keepdim=True))
        s = e / e.sum(1, keepdim=True)
    if st["bias"] is not None:
        choice = s + st["bias"].double()
        score = choice.view(M, G, E // G).sort(dim=-1, descending=True).values[..., :2].sum(-1)
    else:
        choice = x
        score = x.view(M, G, E // G).amax(-1)
    taken = score.sort(dim=-1, descending=True, stable=True).indices[:, :c["topk_group"]]
    alive = torch.zeros(M, G, dtype=torch.bool, device=x.device).scatter_(1, taken, True)
    choice = choice.masked_fill(~alive.repeat_interleave(E // G, 1), -math.inf)
    ids = choice.sort(dim=-1, descending=True, stable=True).indices[:, :c["k"]]
    w = s.gather(1, ids)
    w = w / w.sum(1, keepdim=True) * c["scale"]
    return w.float(), ids.int()


def _values(q, s):
    """f32 values of 1x128-scaled rows."""
    return q.float().view(q.shape[0], -1, BLOCK).mul_(s.unsqueeze(-1)).view(q.shape)


def _weight_values(q, s):
    N, K = q.shape
    rows = s.repeat_interleave(BLOCK, 0)[:N]
    return q.float().view(N, K // BLOCK, BLOCK).mul_(rows.unsqueeze(-1)).view(N, K)


def _plain_product(q, s, w, ws):
    return _values(q, s) @ _weight_values(w, ws).t()


def _plain_gate_up(q, s, w13, w13s):
    y = _plain_product(q, s, w13, w13s)
    gate, up = y[:, 0::2], y[:, 1::2]
    return _quant_rows(gate / (1.0 + torch.exp(-gate)) * up)


def _plain(st):
    c = st["case"]
    if c["op"] == "route":
        return _plain_route(st)
    q, s = (st["x"], st["xs"]) if st["xs"] is not None else _quant_rows(st["x"])
    if c["op"] == "gate_up":
        return _plain_gate_up(q, s, st["w13"], st["w13s"])
    if c["op"] == "linear":
        y = _plain_product(q, s, st["w"], st["ws"])
    else:
        q, s = _plain_gate_up(q, s, st["w13"], st["w13s"])
        y = _plain_product(q, s, st["w2"], st["w2s"])
    if c.get("residual"):
        y = y + st["residual"].float()
    return y if c.get("f32") else y.to(torch.bfloat16)


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _own(st):
    import trials_b200 as fw

    c = st["case"]
    if c["op"] == "route":
        return fw.select_experts(st["logits"], c["k"], c["scoring"], st["bias"], renormalize=True,
                                 routed_scaling_factor=c["scale"], num_expert_group=c["groups"],
                                 topk_group=c["topk_group"])
    if c["op"] == "gate_up":
        return fw.fp8_gate_up(st["x"], st["w13"], st["w13s"], x_scale=st["xs"])
    if c["op"] == "linear":
        return fw.fp8_block_linear(st["x"], st["w"], st["ws"], x_scale=st["xs"], residual=st.get("residual"),
                                   out_dtype=torch.float32 if c["f32"] else torch.bfloat16)
    return fw.fp8_mlp(st["x"], st["w13"], st["w13s"], st["w2"], st["w2s"], residual=st.get("residual"))


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ---------------------------------------------------------------------------
# work and exact values
# ---------------------------------------------------------------------------
def _product_bytes(N, K):
    return N * K + 4 * -(-N // BLOCK) * (K // BLOCK)


def work(case):
    op, M = case["op"], case["M"]
    if op == "route":
        return {"bytes": M * case["E"] * (2 if case["bf16"] else 4) + 8 * M * case["k"],
                "flops": 8 * M * case["E"]}
    K = case["K"] if op == "linear" else case["H"]
    n = case["N"] if op == "linear" else K
    x = M * (K + K // BLOCK * 4 if case.get("quantized") else 2 * K)
    if op == "linear":
        y = M * n * (4 if case["f32"] else 2)
        return {"bytes": x + _product_bytes(n, K) + y + (2 * M * n if case["residual"] else 0),
                "flops": 2 * M * n * K}
    I = case["I"]
    if op == "gate_up":
        return {"bytes": x + _product_bytes(2 * I, K) + M * (I + I // BLOCK * 4), "flops": 4 * M * I * K}
    return {"bytes": x + _product_bytes(2 * I, K) + _product_bytes(K, I) + 2 * M * K * (2 if case["residual"] else 1),
            "flops": 6 * M * I * K}


def _exact_scaled(q, s, rows):
    """64-bit values of codes whose scale covers `rows` rows and 128 columns."""
    n, k = q.shape
    i = torch.arange(n, device=q.device) // rows
    j = torch.arange(k, device=q.device) // BLOCK
    return q.double() * s.double()[i][:, j]


def _exact_input(st):
    """The quantised input as the format defines it (f32 scale and quotient, rounded to e4m3), in 64-bit values."""
    x, s = st["x"], st["xs"]
    if s is None:
        groups = torch.stack(x.float().split(BLOCK, dim=1), dim=1)
        top = groups.abs().max(dim=2).values
        s = torch.maximum(top / torch.full_like(top, 448.0), torch.full_like(top, 1e-12))
        x = torch.cat([(groups[:, j] / s[:, j:j + 1]).clamp(-448.0, 448.0).to(FP8)
                       for j in range(groups.shape[1])], dim=1)
    return _exact_scaled(x, s, 1)


def _exact_gate_up(x, st):
    y = x @ _exact_scaled(st["w13"], st["w13s"], BLOCK).t()
    y = y.view(y.shape[0], -1, 2)
    inter = y[..., 0] * torch.sigmoid(y[..., 0]) * y[..., 1]
    groups = inter.view(inter.shape[0], -1, BLOCK)
    s = torch.maximum(groups.abs().amax(2) / 448.0, torch.tensor(1e-12, dtype=torch.float64, device=y.device))
    q = (groups / s[..., None]).clamp(-448.0, 448.0).to(FP8).double()
    return q.view(inter.shape), s


def _exact_route(st):
    c = st["case"]
    per = c["E"] // c["groups"]
    x = st["logits"].double()
    s = torch.sigmoid(x) if c["scoring"] == "sigmoid" else torch.softmax(x, dim=1)
    left = (s + st["bias"].double() if st["bias"] is not None else x).clone()
    rows = torch.arange(c["M"], device=x.device)
    parts = left.view(c["M"], c["groups"], per)
    score = parts.topk(min(2, per), dim=2).values.sum(2) if st["bias"] is not None else parts.max(2).values
    shut = torch.ones_like(score, dtype=torch.bool)
    for _ in range(c["topk_group"]):  # argmax takes the first of equal values
        best = score.argmax(1)
        shut[rows, best] = False
        score[rows, best] = -math.inf
    parts[shut] = -math.inf
    ids = []
    for _ in range(c["k"]):
        ids.append(left.argmax(1))
        left[rows, ids[-1]] = -math.inf
    w = s.gather(1, torch.stack(ids, 1))
    return w * (c["scale"] / w.sum(1, keepdim=True)), None


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(st)
    x = _exact_input(st)
    if case["op"] == "gate_up":
        return _exact_gate_up(x, st)
    if case["op"] == "linear":
        y = x @ _exact_scaled(st["w"], st["ws"], BLOCK).t()
    else:
        q, s = _exact_gate_up(x, st)
        y = _exact_scaled(q, s, 1) @ _exact_scaled(st["w2"], st["w2s"], BLOCK).t()
    return y + st["residual"].double() if case.get("residual") else y
