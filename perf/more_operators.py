"""The work of linears and routed experts in 8-bit integers with 32-bit scales, and of routed experts in 16-bit values, as cases that can be timed and compared.

Rows in 8 bits: each row (token) has one fp32 scale s = max |x| / 127 and codes q = x / s rounded to the nearest whole number, ties to the even one.  With zero points a row has
s = (high - low) / 255 over low = min(x, 0) and high = max(x, 0), a whole number z = round(-low / s) - 128, and codes round(x / s) + z within [-128, 127]; q stands for (q - z) s.
The scale is at least 2^-100.  Weights have whole numbers in [-127, 127] and one fp32 scale for each output channel.

Five kinds of case, each through the entry points that a program calls:

* `linear`: one projection of 16-bit rows over such weights, `programs.Int8Linear.run`, which quantises the rows;
* `int8 up`: the first products of routed experts, SwiGLU behind them, `programs.Int8MoeLayer.place` and `.up`;
* `int8 down`: their second products and the weighted sum over a token's routes, `.place` and `.down`;
* `half up`, `half down`: the same with weights and rows of fp16 or bf16, `programs.HalfMoeLayer`.
"""
import math

import torch

own = False

LARGEST_PRODUCT = 8192 * 4096 * 4096
LARGEST_MATRIX = 17408 * 5120
LARGEST_BANK = 128 * 2048 * 512
SMALLEST_SCALE = 2.0 ** -100
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    return [
        # one decode row through one small projection: latency counts
        {"name": "linear 1 row", "kind": "linear", "rows": 1, "n": 9728, "k": 2560, "dtype": "bfloat16", "zero_points": False, "bias": False},
        # a batch of decoding requests through a wide projection, rows that are mostly of one sign
        {"name": "linear 32 rows", "kind": "linear", "rows": 32, "n": 17408, "k": 5120, "dtype": "float16", "zero_points": True, "bias": False},
        # a short prompt of ragged length through an attention input projection with biases
        {"name": "linear 333 rows", "kind": "linear", "rows": 333, "n": 7168, "k": 5120, "dtype": "bfloat16", "zero_points": False, "bias": True},
        # a long prompt
        {"name": "linear 8192 rows", "kind": "linear", "rows": 8192, "n": 4096, "k": 4096, "dtype": "bfloat16", "zero_points": True, "bias": True},
        # experts of a decode step of three requests: a few rows of few experts
        {"name": "int8 up 3 tokens", "kind": "int8 up", "tokens": 3, "experts": 128, "top_k": 8, "hidden": 2048, "inner": 512, "dtype": "bfloat16"},
        # a decode batch or a short prompt, some sixteen rows to an expert
        {"name": "int8 down 256 tokens", "kind": "int8 down", "tokens": 256, "experts": 128, "top_k": 8, "hidden": 2048, "inner": 512, "dtype": "bfloat16"},
        # a long prompt
        {"name": "int8 up 4096 tokens", "kind": "int8 up", "tokens": 4096, "experts": 128, "top_k": 8, "hidden": 2048, "inner": 512, "dtype": "bfloat16"},
        {"name": "int8 down 4096 tokens", "kind": "int8 down", "tokens": 4096, "experts": 128, "top_k": 8, "hidden": 2048, "inner": 512, "dtype": "float16"},
        # unquantised experts: the decode step of one request
        {"name": "half up 1 token", "kind": "half up", "tokens": 1, "experts": 128, "top_k": 8, "hidden": 2048, "inner": 512, "dtype": "bfloat16"},
        # few large experts, a short prompt of ragged length
        {"name": "half down 200 tokens", "kind": "half down", "tokens": 200, "experts": 16, "top_k": 2, "hidden": 4096, "inner": 1536, "dtype": "float16"},
        # a long prompt
        {"name": "half up 4096 tokens", "kind": "half up", "tokens": 4096, "experts": 128, "top_k": 8, "hidden": 2048, "inner": 512, "dtype": "bfloat16"},
        {"name": "half down 4096 tokens", "kind": "half down", "tokens": 4096, "experts": 128, "top_k": 8, "hidden": 2048, "inner": 512, "dtype": "bfloat16"},
    ]


def _spread(rng, low, high, step=1):
    """A whole multiple of `step` in [low, high], spread evenly over the logarithm."""
    value = math.exp(rng.uniform(math.log(low), math.log(high + 1)))
    return min(high // step * step, max(-(-low // step) * step, int(value) // step * step))


def draw(rng):
    kind = rng.choice(("linear", "linear", "int8 up", "int8 down", "half up", "half down"))
    dtype = rng.choice(("float16", "bfloat16"))
    if kind == "linear":
        k = _spread(rng, 64, 17408, rng.choice((1, 8, 64)))
        n = _spread(rng, 48, min(17408, LARGEST_MATRIX // k))
        return {"kind": kind, "rows": _spread(rng, 1, min(8192, LARGEST_PRODUCT // (n * k))), "n": n, "k": k, "dtype": dtype,
                "zero_points": rng.random() < 0.5, "bias": rng.random() < 0.5}
    experts = rng.choice((16, 32, 60, 64, 128))
    step = 8 if kind.startswith("half") else rng.choice((1, 8, 32))
    hidden = _spread(rng, 256, 4096, step)
    inner = _spread(rng, 128, max(128, min(1536, LARGEST_BANK // (experts * hidden))), step)
    top_k = rng.choice((1, 2, 4, 6, 8))
    return {"kind": kind, "tokens": _spread(rng, 1, max(1, min(4096, 4096 * 8 * 2048 * 512 // (top_k * hidden * inner)))), "experts": experts, "top_k": top_k,
            "hidden": hidden, "inner": inner, "dtype": dtype}


# ---- the operators in plain operations ----------------------------------------------------------------------------------------------------------
def _quantised_values(x, zero_points):
    """What the codes of rows x (rows, K) stand for, in 32 bits.  (Quotients in 64: those next to a border have to fall on the right side.)"""
    values = x.float()
    if not zero_points:
        scale = (values.abs().amax(1, keepdim=True).double() / 127).float().clamp(min=SMALLEST_SCALE)
        return torch.round(values.double() / scale.double()).float() * scale
    low, high = values.amin(1, keepdim=True).clamp(max=0), values.amax(1, keepdim=True).clamp(min=0)
    scale = ((high - low).double() / 255).float().clamp(min=SMALLEST_SCALE)
    zero = torch.round(-low.double() / scale.double()) - 128
    codes = (torch.round(values.double() / scale.double()) + zero).clamp(-128, 127)
    return (codes - zero).float() * scale


def _silu(x):
    return x / (1 + torch.exp(-x))


# ---- cases --------------------------------------------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(rows, k, dtype, g):
    """Hidden states: normal values, a thousandth of them outliers ten times as large."""
    x = torch.randn((rows, k), generator=g, device="cuda")
    outliers = torch.rand((rows, k), generator=g, device="cuda") < 0.001
    return torch.where(outliers, x * 10, x).to(dtype)


def _stored(weight):
    """Weights (N, K) as they are stored: whole numbers (N, K) and scales (N)."""
    scale = weight.abs().amax(1) / 127
    return torch.round(weight / scale[:, None]).to(torch.int8), scale


def _popularity(experts):
    return [1 / rank ** 1.1 for rank in range(1, experts + 1)]


def _routed(case, g):
    """Distinct experts of every token, popularity like 1 / rank^1.1 in a shuffled order, and weights that sum to one."""
    experts, top_k = case["experts"], case["top_k"]
    order = torch.randperm(experts, generator=g, device="cuda")
    bias = torch.tensor(_popularity(experts), device="cuda").log()[order]
    logits = torch.randn((case["tokens"], experts), generator=g, device="cuda") + bias
    ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :top_k].int().contiguous()
    weight = torch.rand((case["tokens"], top_k), generator=g, device="cuda") + 0.1
    return ids, (weight / weight.sum(1, keepdim=True)).contiguous()


class _Linear:
    def __init__(self, case, seed):
        g = _generator(seed)
        dtype, n, k = DTYPES[case["dtype"]], case["n"], case["k"]
        self.zero_points = case["zero_points"]
        x = _rows(case["rows"], k, torch.float32, g)
        # (zero points are for rows that lie to one side, as behind an activation)
        self.x = (torch.where(x < 0, x * 0.1, x) if self.zero_points else x).to(dtype)
        self.weight, self.scale = _stored(torch.randn((n, k), generator=g, device="cuda") / math.sqrt(k))
        self.bias = torch.randn(n, generator=g, device="cuda") if case["bias"] else None
        if own:
            from orinfer_amd import programs

            self.linear = programs.Int8Linear(self.weight, self.scale, capacity=case["rows"], bias=self.bias, zero_points=self.zero_points, dtype=dtype)

    def run(self):
        if own:
            return self.linear.run(self.x)
        out = _quantised_values(self.x, self.zero_points) @ (self.weight.float() * self.scale[:, None]).t()
        return (out if self.bias is None else out + self.bias).to(self.x.dtype)


class _Experts:
    def __init__(self, case, seed):
        g = _generator(seed)
        self.case, self.int8, self.up = case, case["kind"].startswith("int8"), case["kind"].endswith("up")
        experts, hidden, inner, dtype = case["experts"], case["hidden"], case["inner"], DTYPES[case["dtype"]]
        self.dtype = dtype
        self.ids, self.prob = _routed(case, g)
        if self.up:
            self.x = _rows(case["tokens"], hidden, dtype, g)
        else:  # what the first products leave: products of two normal values, most of them small
            shape = (case["tokens"] * case["top_k"], inner)
            self.act = (_silu(torch.randn(shape, generator=g, device="cuda")) * torch.randn(shape, generator=g, device="cuda")).to(dtype)
        self.gate_up, self.down = self._bank(experts, 2 * inner, hidden, g), self._bank(experts, hidden, inner, g)
        if own:
            from orinfer_amd import programs

            shape = (case["tokens"], experts, case["top_k"], hidden, inner)
            if self.int8:
                self.layer = programs.Int8MoeLayer(*shape, *self.gate_up, *self.down, dtype=dtype)
            else:
                self.layer = programs.HalfMoeLayer(*shape, *self.gate_up, *self.down)

    def _bank(self, experts, n, k, g):
        weight = torch.empty((experts, n, k), dtype=torch.int8 if self.int8 else self.dtype, device="cuda")
        scale = torch.empty((experts, n), device="cuda")
        for e in range(experts):
            values = torch.randn((n, k), generator=g, device="cuda") / math.sqrt(k)
            if self.int8:
                weight[e], scale[e] = _stored(values)
            else:
                weight[e] = values
        return (weight, scale) if self.int8 else (weight,)

    def _weight(self, bank, e):
        return bank[0][e].float() * bank[1][e][:, None] if self.int8 else bank[0][e].float()

    def run(self):
        if own:
            self.layer.place(self.ids)
            return self.layer.up(self.x) if self.up else self.layer.down(self.act, self.prob)
        case = self.case
        order = torch.sort(self.ids.flatten(), stable=True).indices  # assignments in the order of their experts
        counts = torch.bincount(self.ids.flatten(), minlength=case["experts"]).tolist()  # (a plain program asks for the numbers)
        rows = self.x if self.up else self.act
        rows = _quantised_values(rows, False) if self.int8 else rows.float()
        if self.up:
            rows = rows[order // case["top_k"]]
        bank = self.gate_up if self.up else self.down
        parts, first = [], 0
        for e, count in enumerate(counts):
            if count:
                parts.append(rows[first:first + count] @ self._weight(bank, e).t())
                first += count
        products = torch.cat(parts)
        if self.up:
            gate, value = products.chunk(2, dim=1)
            return (_silu(gate) * value).to(self.dtype)
        slot = torch.empty_like(order)
        slot[order] = torch.arange(len(order), device="cuda")
        return (products[slot].view(case["tokens"], case["top_k"], -1) * self.prob[:, :, None]).sum(1).to(self.dtype)


def prepare(case, seed):
    return (_Linear if case["kind"] == "linear" else _Experts)(case, seed)


def run(state):
    return state.run()


def work(case):
    kind = case["kind"]
    if kind == "linear":
        rows, n, k = case["rows"], case["n"], case["k"]
        return {"bytes": n * k + 4 * n + 2 * rows * (n + k) + (4 * n if case["bias"] else 0), "flops": 2 * rows * n * k}
    experts, routes, hidden, inner = case["experts"], case["tokens"] * case["top_k"], case["hidden"], case["inner"]
    popularity = _popularity(experts)
    share = [min(1.0, case["top_k"] * p / sum(popularity)) for p in popularity]
    touched = max(case["top_k"], sum(1 - (1 - s) ** case["tokens"] for s in share))
    n, k = (2 * inner, hidden) if kind.endswith("up") else (hidden, inner)
    weights = n * (k + 4) if kind.startswith("int8") else 2 * n * k
    moved = 2 * (case["tokens"] * hidden + routes * inner) + 4 * routes + (0 if kind.endswith("up") else 4 * routes)
    return {"bytes": int(touched * weights) + moved, "flops": 2 * routes * n * k}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------------------------------
def _exact_rows(x, zero_points):
    """x (rows, K) in 64 bits, each value moved to the nearest one that 8 bits and the row's scale can hold, ties to the even code; the scale is a number of 32 bits."""
    wide = x.double()
    zeros = torch.zeros((len(wide), 1), dtype=torch.float64, device=x.device)
    if zero_points:
        high, low = torch.maximum(wide.max(dim=1, keepdim=True).values, zeros), torch.minimum(wide.min(dim=1, keepdim=True).values, zeros)
        span, levels = (high - low).float().double(), 255
    else:
        high, low = wide.abs().max(dim=1, keepdim=True).values, zeros
        span, levels = high, 127
    step = torch.clamp((span / levels).float(), min=SMALLEST_SCALE).double()
    if not zero_points:
        return torch.round(wide / step) * step
    zero = -128 - torch.round(low / step)
    whole = torch.clamp(torch.round(wide / step) + zero, min=-128, max=127)
    return (whole - zero) * step


def exact(case, seed):
    state, kind = prepare(case, seed), case["kind"]
    if kind == "linear":
        out = torch.mm(_exact_rows(state.x, case["zero_points"]), state.weight.double().t().contiguous()) * state.scale.double()
        return out + state.bias.double() if case["bias"] else out
    up, int8, top_k = kind.endswith("up"), kind.startswith("int8"), case["top_k"]
    ids = state.ids.long()
    rows = state.x if up else state.act
    rows = _exact_rows(rows, False) if int8 else rows.double()
    bank = state.gate_up if up else state.down
    slot_of, first = torch.empty_like(ids), 0  # token-major within an expert
    leaves = torch.empty((ids.numel(), case["inner"] if up else case["hidden"]), dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        token, rank = torch.nonzero(ids == e, as_tuple=True)
        if len(token) == 0:
            continue
        slots = torch.arange(first, first + len(token), device="cuda")
        slot_of[token, rank] = slots
        first += len(token)
        product = torch.mm(rows[token] if up else rows[slots], bank[0][e].double().t().contiguous())
        if int8:
            product = product * bank[1][e].double()
        if up:
            gate, value = product[:, :case["inner"]], product[:, case["inner"]:]
            product = gate * torch.sigmoid(gate) * value
        leaves[slots] = product
    if up:
        return leaves
    out = torch.zeros((case["tokens"], case["hidden"]), dtype=torch.float64, device="cuda")
    for rank in range(top_k):
        out += state.prob[:, rank:rank + 1].double() * leaves[slot_of[:, rank]]
    return out
