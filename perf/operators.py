"""The work of the microscaled 4-bit operators and of the router with scores, balance bias and groups, as cases that can be timed and compared.

MXFP4: a row is cut into blocks of 32 along K; a block has one power of two, stored as its exponent plus 127 in a byte, and 32 codes of one sign, two exponent
and one mantissa bits (0, 0.5, 1, 1.5, 2, 3, 4, 6), two to a byte, the even element in the low half.

Five kinds of case, each through the entry points that a program calls:

* `quantise`: rows of 16-bit values to codes and exponents and back, `lib.Kernel("mxfp4_quantization")` and `lib.Kernel("mxfp4_dequantization")`;
* `linear`: one projection of 16-bit rows over MXFP4 weights, `programs.Mxfp4Linear.run`;
* `up`: the first products of routed experts, SwiGLU behind them, `programs.Mxfp4MoeLayer.place` and `.up`;
* `down`: their second products and the weighted sum over a token's routes, `.place` and `.down`;
* `router`: logits to routes and weights, `lib.Kernel("router_topk")` with its scores, bias and groups.
"""
import math

import torch

own = False

LARGEST_PRODUCT = 8192 * 4096 * 4096
LARGEST_MATRIX = 17408 * 5120
LARGEST_BANK = 128 * 2048 * 512
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BORDERS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)  # between neighbours; a value on one goes to the neighbour with an even code
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    return [
        # a decode batch of odd size, quantised for a projection: the launches are what it costs
        {"name": "quantise 7 rows", "kind": "quantise", "rows": 7, "k": 2560, "dtype": "float16"},
        # the rows of a long prompt
        {"name": "quantise 8192 rows", "kind": "quantise", "rows": 8192, "k": 5120, "dtype": "bfloat16"},
        # one decode row through one small projection
        {"name": "linear 1 row", "kind": "linear", "rows": 1, "n": 9728, "k": 2560, "dtype": "float16"},
        # a batch of decoding requests through a wide projection
        {"name": "linear 32 rows", "kind": "linear", "rows": 32, "n": 17408, "k": 5120, "dtype": "float16"},
        # a short prompt of ragged length through the attention input projection
        {"name": "linear 333 rows", "kind": "linear", "rows": 333, "n": 7168, "k": 5120, "dtype": "bfloat16"},
        # a long prompt
        {"name": "linear 8192 rows", "kind": "linear", "rows": 8192, "n": 4096, "k": 4096, "dtype": "float16"},
        # experts of a decode step of three requests: a few rows of few experts
        {"name": "up 3 tokens", "kind": "up", "tokens": 3, "experts": 128, "top_k": 8, "hidden": 2048, "inner": 512},
        # a decode batch or a short prompt, some sixteen rows to an expert
        {"name": "down 256 tokens", "kind": "down", "tokens": 256, "experts": 128, "top_k": 8, "hidden": 2048, "inner": 512},
        # a long prompt
        {"name": "up 4096 tokens", "kind": "up", "tokens": 4096, "experts": 128, "top_k": 8, "hidden": 2048, "inner": 512},
        {"name": "down 4096 tokens", "kind": "down", "tokens": 4096, "experts": 128, "top_k": 8, "hidden": 2048, "inner": 512},
        # the routes of a decode step: sigmoid scores, a bias for balance, no groups
        {"name": "router 5 tokens", "kind": "router", "tokens": 5, "experts": 128, "top_k": 8, "scoring": "sigmoid", "groups": 1, "top_groups": 1, "scale": 1.0},
        # the routes of a long prompt among the four best of eight groups, weights times 2.5
        {"name": "router 8192 tokens", "kind": "router", "tokens": 8192, "experts": 256, "top_k": 8, "scoring": "sigmoid", "groups": 8, "top_groups": 4, "scale": 2.5},
    ]


def _spread(rng, low, high, step=1):
    """A whole multiple of `step` in [low, high], spread evenly over the logarithm."""
    value = math.exp(rng.uniform(math.log(low), math.log(high + 1)))
    return min(high // step * step, max(-(-low // step) * step, int(value) // step * step))


def draw(rng):
    kind = rng.choice(("quantise", "linear", "linear", "up", "down", "router"))
    if kind == "quantise":
        k = _spread(rng, 32, 17408, rng.choice((1, 8, 32)))
        return {"kind": kind, "rows": _spread(rng, 1, min(8192, 8192 * 5120 // k)), "k": k, "dtype": rng.choice(("float16", "bfloat16"))}
    if kind == "linear":
        k = _spread(rng, 64, 17408, 32)
        n = _spread(rng, 48, min(17408, LARGEST_MATRIX // k))
        return {"kind": kind, "rows": _spread(rng, 1, min(8192, LARGEST_PRODUCT // (n * k))), "n": n, "k": k, "dtype": rng.choice(("float16", "bfloat16"))}
    if kind == "router":
        groups = rng.choice((1, 1, 2, 4, 8))
        size = _spread(rng, 8, 512 // groups)
        top_groups = rng.randint(1, groups)
        return {"kind": kind, "tokens": _spread(rng, 1, 8192 * 256 // (groups * size)), "experts": groups * size, "top_k": rng.randint(1, 8),
                "scoring": rng.choice(("sigmoid", "softmax")), "groups": groups, "top_groups": top_groups, "scale": rng.choice((1.0, 2.5))}
    experts = rng.choice((16, 32, 60, 64, 128))
    hidden = _spread(rng, 256, 4096, 32)
    inner = _spread(rng, 128, max(128, min(1536, LARGEST_BANK // (experts * hidden))), 32)
    top_k = rng.choice((1, 2, 4, 6, 8))
    return {"kind": kind, "tokens": _spread(rng, 1, max(1, min(4096, 4096 * 8 * 2048 * 512 // (top_k * hidden * inner)))), "experts": experts, "top_k": top_k,
            "hidden": hidden, "inner": inner}


# ---- the format in plain operations -----------------------------------------------------------------------------------------------------------
def _quantised_values(x):
    """The values that a row's codes stand for, in 32 bits: x (rows, K) of any type; a last block may be short."""
    rows, k = x.shape
    values = torch.nn.functional.pad(x.float(), (0, -k % 32)).view(rows, -1, 32)
    largest = values.abs().amax(-1, keepdim=True)
    exponent = (largest.view(torch.int32) >> 23) - 2  # of the largest's power of two, plus 127, minus the two that the largest code has
    power = torch.ldexp(torch.ones_like(largest), exponent.clamp(min=0) - 127)
    scaled = values / power
    magnitude = scaled.abs()
    found = torch.zeros_like(magnitude)
    for i, border in enumerate(BORDERS):  # the upper neighbour's code is i + 1: a value on the border goes up where that is even
        above = magnitude >= border if i % 2 else magnitude > border
        found = torch.where(above, torch.full_like(found, MAGNITUDES[i + 1]), found)
    return (torch.copysign(found, scaled) * power).reshape(rows, -1)[:, :k]


def _stored(values):
    """Weights (..., K) as they are stored: codes (..., K / 2) and exponents (..., K / 32)."""
    blocks = values.unflatten(-1, (-1, 32))
    largest = blocks.abs().amax(-1, keepdim=True)
    exponent = ((largest.view(torch.int32) >> 23) - 2).clamp(min=0)
    scaled = blocks * torch.ldexp(torch.ones_like(largest), 127 - exponent)
    magnitude = scaled.abs()
    code = torch.zeros_like(magnitude, dtype=torch.uint8)
    for i, border in enumerate(BORDERS):
        code += (magnitude >= border if i % 2 else magnitude > border).to(torch.uint8)
    code += 8 * torch.signbit(scaled).to(torch.uint8)
    code = code.flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), exponent.squeeze(-1).to(torch.uint8)


def _stored_values(codes, exponents):
    """What stored weights (N, K / 2) stand for, (N, K) in 32 bits."""
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=codes.device)
    both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    power = torch.ldexp(torch.ones((), device=codes.device), exponents.int() - 127)
    return table[both.int()] * power.repeat_interleave(32, -1)


def _silu(x):
    return x / (1 + torch.exp(-x))


# ---- cases ------------------------------------------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(case, rows, k, dtype, g):
    """Hidden states: normal values, a thousandth of them outliers twenty times as large."""
    x = torch.randn((rows, k), generator=g, device="cuda")
    outliers = torch.rand((rows, k), generator=g, device="cuda") < 0.001
    return torch.where(outliers, x * 20, x).to(dtype)


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


def _expert_weights(case, g):
    experts, hidden, inner = case["experts"], case["hidden"], case["inner"]

    def bank(n, k):
        codes = torch.empty((experts, n, k // 2), dtype=torch.uint8, device="cuda")
        exponents = torch.empty((experts, n, k // 32), dtype=torch.uint8, device="cuda")
        for e in range(experts):
            codes[e], exponents[e] = _stored(torch.randn((n, k), generator=g, device="cuda") / math.sqrt(k))
        return codes, exponents

    return bank(2 * inner, hidden), bank(hidden, inner)


class _Quantise:
    def __init__(self, case, seed):
        self.rows, self.k = case["rows"], case["k"]
        self.x = _rows(case, self.rows, self.k, DTYPES[case["dtype"]], _generator(seed))
        if own:
            from orinfer_amd import lib

            blocks = -(-self.k // 32)
            self.q = torch.empty((self.rows, blocks * 16), dtype=torch.uint8, device="cuda")
            self.s = torch.empty((self.rows, blocks), dtype=torch.uint8, device="cuda")
            self.values = torch.empty_like(self.x)
            self.quantise = lib.Kernel("mxfp4_quantization", K=self.k, input_dtype=case["dtype"])
            self.dequantise = lib.Kernel("mxfp4_dequantization", K=self.k, output_dtype=case["dtype"])

    def run(self):
        if own:
            self.quantise(Q=self.q, S=self.s, X=self.x, rows=self.rows)
            self.dequantise(Q=self.q, S=self.s, Y=self.values, rows=self.rows)
            return self.values
        return _quantised_values(self.x).to(self.x.dtype)


class _Linear:
    def __init__(self, case, seed):
        g = _generator(seed)
        self.x = _rows(case, case["rows"], case["k"], DTYPES[case["dtype"]], g)
        self.codes, self.exponents = _stored(torch.randn((case["n"], case["k"]), generator=g, device="cuda") / math.sqrt(case["k"]))
        if own:
            from orinfer_amd import programs

            self.linear = programs.Mxfp4Linear(self.codes, self.exponents, capacity=case["rows"], dtype=self.x.dtype)

    def run(self):
        if own:
            return self.linear.run(self.x)
        return (_quantised_values(self.x) @ _stored_values(self.codes, self.exponents).t()).to(self.x.dtype)


class _Experts:
    def __init__(self, case, seed):
        g = _generator(seed)
        self.case = case
        self.ids, self.prob = _routed(case, g)
        if case["kind"] == "up":
            self.x = _rows(case, case["tokens"], case["hidden"], torch.float16, g)
        else:  # what the first products leave: products of two normal values, most of them small
            shape = (case["tokens"] * case["top_k"], case["inner"])
            self.act = (_silu(torch.randn(shape, generator=g, device="cuda")) * torch.randn(shape, generator=g, device="cuda")).to(torch.float16)
        self.gate_up, self.down = _expert_weights(case, g)
        if own:
            from orinfer_amd import programs

            self.layer = programs.Mxfp4MoeLayer(case["tokens"], case["experts"], case["top_k"], case["hidden"], case["inner"], *self.gate_up, *self.down)

    def _places(self):
        """Assignments in the order of their experts, and how many each expert has (a plain program asks for the numbers)."""
        order = torch.sort(self.ids.flatten(), stable=True).indices
        return order, torch.bincount(self.ids.flatten(), minlength=self.case["experts"]).tolist()

    def run(self):
        up = self.case["kind"] == "up"
        if own:
            self.layer.place(self.ids)
            return self.layer.up(self.x) if up else self.layer.down(self.act, self.prob)
        order, counts = self._places()
        rows = _quantised_values(self.x)[order // self.case["top_k"]] if up else _quantised_values(self.act)
        codes, exponents = self.gate_up if up else self.down
        parts, first = [], 0
        for e, count in enumerate(counts):
            if count:
                parts.append(rows[first:first + count] @ _stored_values(codes[e], exponents[e]).t())
                first += count
        products = torch.cat(parts)
        if up:
            gate, value = products.chunk(2, dim=1)
            return (_silu(gate) * value).to(torch.float16)
        slot = torch.empty_like(order)
        slot[order] = torch.arange(len(order), device="cuda")
        return (products[slot].view(self.case["tokens"], self.case["top_k"], -1) * self.prob[:, :, None]).sum(1).to(torch.float16)


class _Router:
    def __init__(self, case, seed):
        g = _generator(seed)
        self.case = case
        experts = case["experts"]
        skew = torch.tensor(_popularity(experts), device="cuda").log()[torch.randperm(experts, generator=g, device="cuda")]
        self.logits = torch.randn((case["tokens"], experts), generator=g, device="cuda") * 1.5 + 0.3 * skew
        # a bias that a balancing rule has moved by small steps
        self.bias = torch.randn(experts, generator=g, device="cuda") * (0.05 if case["scoring"] == "sigmoid" else 0.005)
        if own:
            from orinfer_amd import lib

            self.ids = torch.empty((case["tokens"], case["top_k"]), dtype=torch.int32, device="cuda")
            self.prob = torch.empty((case["tokens"], case["top_k"]), dtype=torch.float32, device="cuda")
            self.router = lib.Kernel("router_topk", M=case["tokens"], E=experts, top_k=case["top_k"], scoring=case["scoring"], bias=True,
                                     groups=case["groups"], top_groups=case["top_groups"], scale=case["scale"])

    def run(self):
        if own:
            self.router(Bias=self.bias, IDs=self.ids, Logits=self.logits, Prob=self.prob)
            return self.ids, self.prob
        case = self.case
        logits = self.logits.double()  # scores next to one another are told apart
        if case["scoring"] == "sigmoid":
            score = 1 / (1 + torch.exp(-logits))
        else:
            score = torch.exp(logits - logits.amax(1, keepdim=True))
            score = score / score.sum(1, keepdim=True)
        choice = score + self.bias.double()
        groups = choice.view(case["tokens"], case["groups"], -1)
        best_two = torch.sort(groups, dim=2, descending=True).values[:, :, :2].sum(2)
        kept = torch.sort(best_two, dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        closed = torch.ones_like(best_two, dtype=torch.bool).scatter_(1, kept, False)
        choice = groups.masked_fill(closed[:, :, None], -math.inf).view_as(choice)
        ids = torch.sort(choice, dim=1, descending=True, stable=True).indices[:, :case["top_k"]]
        weight = score.gather(1, ids)
        weight = weight / weight.sum(1, keepdim=True) * case["scale"]
        return ids.int(), weight.float()


def prepare(case, seed):
    return {"quantise": _Quantise, "linear": _Linear, "up": _Experts, "down": _Experts, "router": _Router}[case["kind"]](case, seed)


def run(state):
    return state.run()


def work(case):
    kind = case["kind"]
    if kind == "quantise":
        count = case["rows"] * case["k"]
        return {"bytes": 4 * count, "flops": 2 * count}
    if kind == "linear":
        rows, n, k = case["rows"], case["n"], case["k"]
        return {"bytes": n * k * 17 // 32 + 2 * rows * (n + k), "flops": 2 * rows * n * k}
    if kind == "router":
        return {"bytes": case["tokens"] * (4 * case["experts"] + 8 * case["top_k"]) + 4 * case["experts"], "flops": 4 * case["tokens"] * case["experts"]}
    experts, routes, hidden, inner = case["experts"], case["tokens"] * case["top_k"], case["hidden"], case["inner"]
    popularity = _popularity(experts)
    share = [min(1.0, case["top_k"] * p / sum(popularity)) for p in popularity]
    touched = max(case["top_k"], sum(1 - (1 - s) ** case["tokens"] for s in share))
    n, k = (2 * inner, hidden) if kind == "up" else (hidden, inner)
    moved = 2 * (case["tokens"] * hidden + routes * inner) + 4 * routes + (4 * routes if kind == "down" else 0)
    return {"bytes": int(touched * n * k * 17 / 32) + moved, "flops": 2 * routes * n * k}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------------------------------
def _exact_rows(x):
    """x (rows, K) in 64 bits, each block of 32 rounded to the nearest value that four bits and its power of two can hold, ties to the even code."""
    rows, k = x.shape
    wide = torch.zeros((rows, -(-k // 32) * 32), dtype=torch.float64, device=x.device)
    wide[:, :k] = x.double()
    wide = wide.view(rows, -1, 32)
    largest = wide.abs().max(dim=2, keepdim=True).values
    power = torch.frexp(largest).exponent - 1 - 2  # largest = m 2^e with m in [1/2, 1)
    power = torch.where(largest == 0, torch.full_like(power, -127), power.clamp(min=-127))
    unit = torch.ldexp(torch.ones_like(largest), power)
    size = (wide.abs() / unit).clamp(max=6.0)
    # the distance between neighbours is 1/2 below 2, 1 below 4 and 2 above
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0)).double()
    return (torch.sign(wide) * torch.round(size / step) * step * unit).view(rows, -1)[:, :k]


def _exact_weights(codes, exponents):
    n = codes.shape[0]
    nibble = torch.empty((n, codes.shape[1] * 2), dtype=torch.int64, device=codes.device)
    nibble[:, 0::2] = (codes % 16).long()
    nibble[:, 1::2] = (codes // 16).long()
    sign, high, low = 1 - 2 * (nibble // 8), nibble % 8 // 2, nibble % 2
    size = torch.where(high == 0, low * 0.5, (1 + low * 0.5) * 2.0 ** (high - 1).double())
    return (sign * size).view(n, -1, 32).mul(2.0 ** (exponents.double() - 127)[:, :, None]).view(n, -1)


def exact(case, seed):
    state, kind = prepare(case, seed), case["kind"]
    if kind == "quantise":
        return _exact_rows(state.x)
    if kind == "linear":
        return torch.mm(_exact_rows(state.x), _exact_weights(state.codes, state.exponents).t().contiguous())
    if kind == "router":
        return _exact_routes(case, state)
    up, top_k = kind == "up", case["top_k"]
    ids = state.ids.long()
    rows = _exact_rows(state.x if up else state.act)
    slot_of, first = torch.empty_like(ids), 0  # token-major within an expert
    leaves = torch.empty((ids.numel(), case["inner"] if up else case["hidden"]), dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        token, rank = torch.nonzero(ids == e, as_tuple=True)
        if len(token) == 0:
            continue
        slots = torch.arange(first, first + len(token), device="cuda")
        slot_of[token, rank] = slots
        first += len(token)
        mine = rows[token] if up else rows[slots]
        product = torch.mm(mine, _exact_weights(*(bank[e] for bank in (state.gate_up if up else state.down))).t().contiguous())
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


def _exact_routes(case, state):
    logits, bias = state.logits.double(), state.bias.double()
    score = torch.sigmoid(logits) if case["scoring"] == "sigmoid" else torch.softmax(logits, dim=1)
    tokens, experts = logits.shape
    size = experts // case["groups"]
    choice = score + bias
    group_score = torch.stack([choice[:, g * size:(g + 1) * size].topk(min(2, size), dim=1).values.sum(1) for g in range(case["groups"])], dim=1)
    left = torch.full_like(choice, -math.inf)
    row = torch.arange(tokens, device="cuda")
    group_of = torch.arange(experts, device="cuda") // size
    for _ in range(case["top_groups"]):
        best = (group_score == group_score.max(dim=1, keepdim=True).values).long().argmax(dim=1)  # the first of equals
        group_score[row, best] = -math.inf
        left = torch.where(group_of[None] == best[:, None], choice, left)
    ids = torch.empty((tokens, case["top_k"]), dtype=torch.int64, device="cuda")
    for rank in range(case["top_k"]):
        ids[:, rank] = (left == left.max(dim=1, keepdim=True).values).long().argmax(dim=1)
        left[row, ids[:, rank]] = -math.inf
    weight = score[row[:, None], ids]
    return ids.int(), weight / weight.sum(dim=1, keepdim=True) * case["scale"]
