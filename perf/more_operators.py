"""Cases of the grouped operators: linear layers whose rows belong to experts or carry
low-rank adapters, on FP8 block products, and the grouping of rows that both start from.

Operators and the public calls they are reached through:

  group    sr_states.group_rows(index, groups)            rows in the order of their groups
  expert   sr_states.expert_linear(x, weight, ends)       y = x W_e^T for the rows of expert e: forward
                                                          and both gradients, or forward on kept blocks
  adapter  sr_states.adapter_linear(x, weight, down, up, groups, scale=s)
                                                          y = x W^T + s_a (x A_a^T) B_a^T for rows of
                                                          adapter a: forward and the gradients of x, A
                                                          and B, or forward alone

``run`` computes the plain form with elementary torch operations in FP32, or
with ``own`` the framework's call.  ``exact`` computes the same outputs in FP64.
"""

import math
import random
import sys

import torch

own = False

_PACKAGE = "stochastic-rounding-pytorch_b200"
_BLOCK = 128
_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16,
           "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
# Largest value, mantissa bits and exponent of the smallest normal number.
_GRID = {"e4m3": (448.0, 3, -6), "e5m2": (57344.0, 2, -14)}
_M32 = 0xFFFFFFFF
_SEED = 5


def _package():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    import sr_states

    return sr_states


# ------------------------------------------------------------------- cases --


def listed():
    return [
        # 8 decoded tokens sent to 2 of 8 experts each: launch latency
        {"name": "group-16-of-8", "op": "group", "rows": 16, "groups": 8, "none": 0},
        # a batch of 8192 tokens sent to 8 of 64 experts each, some of them dropped
        {"name": "group-65536-of-64", "op": "group", "rows": 65536, "groups": 64, "none": 777},
        # one decoded token through 2 of 8 experts with a Llama-3-8B up projection each
        {"name": "expert-serve-2-of-8-4096x14336", "op": "expert", "rows": 2, "experts": 8,
         "active": 2, "tail": 0, "k": 4096, "n": 14336, "dtype": "bf16", "grad": "e4m3",
         "train": False},
        # 32 decoded tokens through 8 of 64 small experts each
        {"name": "expert-serve-256-of-64-2048x1024", "op": "expert", "rows": 256, "experts": 64,
         "active": 62, "tail": 0, "k": 2048, "n": 1024, "dtype": "bf16", "grad": "e4m3",
         "train": False},
        # a prompt of 4096 tokens through 2 of 8 experts each, down projection
        {"name": "expert-serve-8192-of-8-14336x4096", "op": "expert", "rows": 8192, "experts": 8,
         "active": 8, "tail": 0, "k": 14336, "n": 4096, "dtype": "bf16", "grad": "e4m3",
         "train": False},
        # a training step of odd sizes: an expert without rows, rows behind the last expert's
        {"name": "expert-train-1000-of-5-333x777", "op": "expert", "rows": 1000, "experts": 5,
         "active": 4, "tail": 24, "k": 333, "n": 777, "dtype": "f32", "grad": "e5m2",
         "train": True},
        # a training step of 4096 tokens through 2 of 8 experts each, up projection
        {"name": "expert-train-8192-of-8-4096x14336", "op": "expert", "rows": 8192, "experts": 8,
         "active": 8, "tail": 0, "k": 4096, "n": 14336, "dtype": "bf16", "grad": "e4m3",
         "train": True},
        # one decoded token of one request beside a Llama-3-8B attention projection
        {"name": "adapter-serve-1-4096x4096-r16", "op": "adapter", "tokens": 1, "adapters": 8,
         "active": 1, "none": 0, "rank": 16, "k": 4096, "n": 4096, "order": "mixed",
         "dtype": "bf16", "train": False},
        # one decoded token each of 64 requests, most with an adapter of their own
        {"name": "adapter-serve-64-of-48-4096x14336-r16", "op": "adapter", "tokens": 64,
         "adapters": 48, "active": 40, "none": 6, "rank": 16, "k": 4096, "n": 14336,
         "order": "mixed", "dtype": "bf16", "train": False},
        # prompts of 16 requests in one batch
        {"name": "adapter-serve-4096-of-32-4096x4096-r64", "op": "adapter", "tokens": 4096,
         "adapters": 32, "active": 16, "none": 100, "rank": 64, "k": 4096, "n": 4096,
         "order": "runs", "dtype": "bf16", "train": False},
        # a training step of odd sizes, tokens of 7 adapters in any order
        {"name": "adapter-train-500-of-7-1111x777-r12", "op": "adapter", "tokens": 500,
         "adapters": 7, "active": 6, "none": 11, "rank": 12, "k": 1111, "n": 777,
         "order": "mixed", "dtype": "f16", "train": True},
        # a training step of 4 adapters at once on a frozen Llama-3-8B up projection
        {"name": "adapter-train-4096-of-4-4096x14336-r16", "op": "adapter", "tokens": 4096,
         "adapters": 4, "active": 4, "none": 0, "rank": 16, "k": 4096, "n": 14336,
         "order": "runs", "dtype": "bf16", "train": True},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _odd(rng, size):
    """A size near `size`: half of the time a multiple of 128 or of 16, else as drawn."""
    step = rng.choice((1, 1, 16, 128))
    return max(step, size // step * step)


def draw(rng):
    op = rng.choice(("group", "expert", "expert", "adapter", "adapter"))
    if op == "group":
        rows = _log(rng, 1, 65536)
        return {"op": op, "rows": rows, "groups": _log(rng, 1, 256),
                "none": rng.choice((0, rows // 10, rng.randint(0, rows)))}
    train = rng.random() < 0.5
    k, n = _odd(rng, _log(rng, 64, 4096)), _odd(rng, _log(rng, 64, 8192))
    if op == "expert":
        experts = _log(rng, 1, 64)
        most = max(1, int(2.5e8 / (k * n)))  # the weights of the largest listed case, halved
        experts = min(experts, most)
        rows = _log(rng, 1, 8192)
        return {"op": op, "rows": rows, "experts": experts,
                "active": rng.randint(1, min(rows, experts)),
                "tail": rng.choice((0, 0, rng.randint(1, 300))), "k": k, "n": n,
                "dtype": rng.choice(("bf16", "bf16", "f16", "f32")),
                "grad": rng.choice(("e4m3", "e5m2")), "train": train}
    adapters, tokens = _log(rng, 1, 64), _log(rng, 1, 4096)
    none = rng.choice((0, 0, tokens // 8))
    return {"op": op, "tokens": tokens, "adapters": adapters,
            "active": rng.randint(1, min(tokens - none, adapters)), "none": none,
            "rank": rng.choice((4, 8, 12, 16, 32, 64, _log(rng, 1, 128))), "k": k, "n": n,
            "order": rng.choice(("mixed", "runs")), "dtype": rng.choice(("bf16", "f16")),
            "train": train}


def work(case):
    size = {name: torch.empty((), dtype=v).element_size() for name, v in _DTYPES.items()}
    op = case["op"]
    if op == "group":
        return {"bytes": 4 * (2 * case["rows"] + case["groups"]), "flops": 0}
    k, n, each = case["k"], case["n"], size[case["dtype"]]
    if op == "expert":
        t = case["rows"]
        if not case["train"]:
            return {"bytes": case["active"] * n * k + each * (t * (k + n) + case["tail"] * n),
                    "flops": 2.0 * t * k * n}
        weights = each * n * k * (case["active"] + case["experts"])
        return {"bytes": weights + 2 * each * ((t + case["tail"]) * (k + n)),
                "flops": 6.0 * t * k * n}
    t, low = case["tokens"], (case["tokens"] - case["none"]) * case["rank"] * (k + n)
    matrices = each * case["rank"] * (k + n)
    if not case["train"]:
        return {"bytes": n * k + case["active"] * matrices + each * t * (k + n),
                "flops": 2.0 * t * k * n + 2.0 * low}
    return {"bytes": 2 * n * k + (case["active"] + case["adapters"]) * matrices
            + 2 * each * t * (k + n),
            "flops": 4.0 * t * k * n + 6.0 * low}


# ------------------------------------------------------------------ inputs --


def _activations(gen, rows, cols):
    """Rows of different sizes and a few channels far above the rest, as activations have."""
    x = torch.randn((rows, cols), generator=gen, device="cuda")
    x *= torch.exp(0.5 * torch.randn((rows, 1), generator=gen, device="cuda"))
    x *= torch.exp(0.7 * torch.randn((1, cols), generator=gen, device="cuda"))
    return x


def _gradient(gen, rows, cols):
    """Noise, and as much energy in a few directions."""
    x = torch.randn((rows, cols), generator=gen, device="cuda")
    left = torch.randn((rows, 8), generator=gen, device="cuda")
    right = torch.randn((8, cols), generator=gen, device="cuda")
    return (x + 0.35 * (left @ right)) * 1e-4


def _sizes(rng, rows, groups, active):
    """How many rows each group has: `active` of them at least one, uneven as routers are."""
    chosen = rng.sample(range(groups), active)
    share = [math.exp(rng.gauss(0.0, 0.7)) for _ in chosen]
    sizes = [0] * groups
    for g in chosen:
        sizes[g] = 1
    for g in rng.choices(chosen, weights=share, k=rows - active):
        sizes[g] += 1
    return sizes


def _plan(index, groups):
    """(order, ends): rows in the order of their groups, others behind."""
    kept = [i if 0 <= i < groups else groups for i in index]
    order = sorted(range(len(kept)), key=kept.__getitem__)
    count = [0] * (groups + 1)
    for i in kept:
        count[i] += 1
    ends, total = [], 0
    for c in count[:groups]:
        total += c
        ends.append(total)
    return order, ends


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    op, state = case["op"], {"case": case, "seed": seed}
    if op == "group":
        rows, groups = case["rows"], case["groups"]
        weights = [math.exp(rng.gauss(0.0, 0.7)) for _ in range(groups)]
        index = rng.choices(range(groups), weights=weights, k=rows)
        for i in rng.sample(range(rows), case["none"]):
            index[i] = -1
        state["index"] = _ints(index)
        return state
    k, n, dtype = case["k"], case["n"], _DTYPES[case["dtype"]]
    rows = case["rows"] + case["tail"] if op == "expert" else case["tokens"]
    state["x"] = _activations(gen, rows, k).to(dtype)
    if case["train"]:
        state["x"].requires_grad_()
        state["dy"] = _gradient(gen, rows, n).to(dtype)
    if op == "expert":
        state["sizes"] = _sizes(rng, case["rows"], case["experts"], case["active"])
        ends, total = [], 0
        for size in state["sizes"]:
            total += size
            ends.append(total)
        state["ends"] = _ints(ends)
        w = torch.randn((case["experts"], n, k), generator=gen, device="cuda") * 0.02
        if case["train"]:
            state["w"] = w.to(dtype).requires_grad_()
        else:
            # a server keeps its experts in FP8 with one scale a 128 x 128 block
            both = [_quantize(v, "e4m3", "nearest", "square", 0) for v in w]
            state["w"] = tuple(torch.stack([b[i].view(torch.uint8) for b in both])
                               for i in range(2))
            state["w"] = (state["w"][0].view(_DTYPES["e4m3"]), state["w"][1])
        return state
    sizes = _sizes(rng, case["tokens"] - case["none"], case["adapters"], case["active"])
    runs = [[a] * size for a, size in enumerate(sizes)] + [[-1] * case["none"]]
    rng.shuffle(runs)
    index = [a for run in runs for a in run]
    if case["order"] == "mixed":
        rng.shuffle(index)
    order, ends = _plan(index, case["adapters"])
    # the plan of the batch, made once for all layers that its tokens go through
    state["index"], state["plan"] = _ints(index), (_ints(order), _ints(ends))
    state["sizes"] = sizes
    rank, many = case["rank"], case["adapters"]
    down = torch.randn((many, rank, k), generator=gen, device="cuda") * k ** -0.5
    up = torch.randn((many, n, rank), generator=gen, device="cuda") * 0.02
    state["down"], state["up"] = down.to(dtype), up.to(dtype)
    state["scale"] = torch.rand((many,), generator=gen, device="cuda") + 0.5
    w = torch.randn((n, k), generator=gen, device="cuda") * 0.02
    # the shared projection is kept in FP8 blocks, for both directions where it trains
    state["w"] = _quantize(w, "e4m3", "nearest", "square", 0)
    if case["train"]:
        state["down"].requires_grad_(), state["up"].requires_grad_()
        state["w_t"] = _quantize(w.t().contiguous(), "e4m3", "nearest", "square", 0)
    return state


# -------------------------------------------------------------- plain forms --


def _h32(x):
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & _M32
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & _M32
    return x ^ (x >> 16)


def _key(seed, index):
    """Counter base of stored copy `index` under `seed` (a host integer)."""
    return int(_h32(torch.tensor((seed ^ index) & _M32, dtype=torch.int64)))


def _pow2(k):
    """2^k in FP32 for whole k from -127 to 127, from its encoding."""
    k = k.to(torch.int32)
    return torch.where(k > -127, (k + 127) << 23, torch.full_like(k, 1 << 22)).view(torch.float32)


def _round(y, name, rounding, key):
    """FP32 `y` to the named 8-bit type, saturating; `key`: counter of its first element."""
    most, mantissa, low = _GRID[name]
    y = torch.where(torch.isnan(y), y, y.clamp(-most, most))
    if rounding == "nearest":
        return y.to(_DTYPES[name])
    flat = torch.arange(y.numel(), device=y.device).view(y.shape)
    hashes = _h32((flat + key) & _M32)
    exponent = (((y.view(torch.int32) >> 23) & 0xFF) - 127).clamp(min=low)
    unit = _pow2(exponent - mantissa)
    steps = y.abs() / unit
    whole = steps.floor()
    threshold = ((steps - whole) * 16777216.0).floor().to(torch.int64)
    up = ((hashes >> 8) < threshold).to(torch.float32)
    return torch.copysign((whole + up) * unit, y).to(_DTYPES[name])


def _quantize(x, name, rounding, block, key, transposed=False):
    """(data, exponent + 127) of a tensor in blocks of 128 along its last dimension;
    `transposed`: of x.T, with the counters of x."""
    x = x.float()
    if transposed:
        x = x.t()
    square = block == "square"
    rows, cols = x.shape
    high = _BLOCK if square else 1
    view = torch.nn.functional.pad(x, (0, -cols % _BLOCK, 0, -rows % high))
    view = view.view(view.shape[0] // high, high, view.shape[1] // _BLOCK, _BLOCK)
    size = torch.where(torch.isfinite(view), view.abs(), torch.zeros_like(view))
    top = size.amax(dim=(1, 3), keepdim=True)
    fraction, exponent = torch.frexp(top)  # top = fraction * 2^exponent, 0.5 <= fraction < 1
    ceiling = 9 if name == "e4m3" else 16  # the largest value is 0.875 * 2^ceiling
    k = exponent - ceiling + (fraction > 0.875).to(exponent.dtype)
    k = torch.where(top == 0, torch.zeros_like(k), k.clamp(min=-127))
    scaled = (view * _pow2(-k)).view(view.shape[0] * view.shape[1], -1)
    scaled = scaled[:rows, :cols]
    if transposed:
        data = _round(scaled.t().contiguous(), name, rounding, key).t().contiguous()
    else:
        data = _round(scaled.contiguous(), name, rounding, key)
    return data, (k + 127).to(torch.uint8).view(k.shape[0], k.shape[2])


def _values(data, scale):
    """FP32 values of a quantised matrix."""
    rows, cols = data.shape
    factor = _pow2(scale.to(torch.int32) - 127).repeat_interleave(_BLOCK, 1)[:, :cols]
    if scale.shape[0] != rows:
        factor = factor.repeat_interleave(_BLOCK, 0)[:rows]
    return data.float() * factor


def _plain_group(state):
    index, groups = state["index"].long(), state["case"]["groups"]
    kept = torch.where((index >= 0) & (index < groups), index, torch.full_like(index, groups))
    order = torch.sort(kept, stable=True).indices
    # added one by one on purpose: counts are whole numbers, their order does not matter
    count = torch.zeros(groups + 1, dtype=torch.int64, device=index.device)
    count.index_add_(0, kept, torch.ones_like(kept))
    return order.to(torch.int32), count[:groups].cumsum(0).to(torch.int32)


def _plain_expert(state):
    case, x = state["case"], state["x"].detach()
    dtype, train = x.dtype, case["train"]
    values = _values(*_quantize(x, "e4m3", "nearest", "row", 0))
    y = torch.zeros((x.shape[0], case["n"]), device=x.device)
    if train:
        dy, grad = state["dy"], case["grad"]
        row_key, column_key = _key(_SEED, 0), _key(_SEED, 1)
        rows = _values(*_quantize(dy, grad, "stochastic", "row", row_key))
        dx = torch.zeros(x.shape, device=x.device)
        dw = torch.zeros(state["w"].shape, device=x.device)
    start = 0
    for e, size in enumerate(state["sizes"]):
        end = start + size
        if size == 0:
            continue
        if not train:
            w = _values(state["w"][0][e], state["w"][1][e])
            y[start:end] = values[start:end] @ w.t()
        else:
            w = _values(*_quantize(state["w"].detach()[e], "e4m3", "nearest", "square", 0))
            y[start:end] = values[start:end] @ w.t()
            dx[start:end] = rows[start:end] @ w
            columns = _values(*_quantize(dy[start:end], grad, "stochastic", "row",
                                         column_key + start * case["n"], True))
            tokens = _values(*_quantize(x[start:end], "e4m3", "nearest", "row", 0, True))
            dw[e] = columns @ tokens.t()
        start = end
    return (y.to(dtype), dx.to(dtype), dw.to(dtype)) if train else y.to(dtype)


def _plain_adapter(state):
    case, x = state["case"], state["x"].detach()
    dtype, train = x.dtype, case["train"]
    order, scale = state["plan"][0].long(), state["scale"]
    down, up = state["down"].detach(), state["up"].detach()
    y = _values(*_quantize(x, "e4m3", "nearest", "row", 0)) @ _values(*state["w"]).t()
    if train:
        dy = state["dy"]
        dx = (_values(*_quantize(dy, "e4m3", "stochastic", "row", _key(_SEED, 0)))
              @ _values(*state["w_t"]).t())
        ddown = torch.zeros(down.shape, device=x.device)
        dup = torch.zeros(up.shape, device=x.device)
    start = 0
    for a, size in enumerate(state["sizes"]):
        if size == 0:
            continue
        rows = order[start:start + size]
        start += size
        xa, da, ua = x[rows].float(), down[a].float(), up[a].float()
        low = scale[a] * (xa @ da.t())
        y[rows] += low @ ua.t()
        if train:
            g = dy[rows].float()
            back = scale[a] * (g @ ua)
            dx[rows] += back @ da
            ddown[a] = back.t() @ xa
            dup[a] = g.t() @ low
    if not train:
        return y.to(dtype)
    return y.to(dtype), dx.to(dtype), ddown.to(dtype), dup.to(dtype)


_PLAIN = {"group": _plain_group, "expert": _plain_expert, "adapter": _plain_adapter}


# --------------------------------------------------------------------- run --


def _blocks(sr, held):
    return sr.BlockTensor(held[0], held[1].view(torch.float8_e8m0fnu))


def _framework(state):
    sr = _package()
    case, op = state["case"], state["case"]["op"]
    if op == "group":
        got = sr.group_rows(state["index"], case["groups"])
        return got.order, got.ends
    if op == "expert":
        if not case["train"]:
            return sr.expert_linear(state["x"], _blocks(sr, state["w"]), state["ends"])
        y = sr.expert_linear(state["x"], state["w"], state["ends"],
                             grad_dtype=_DTYPES[case["grad"]], seed=_SEED)
        return (y.detach(), *torch.autograd.grad(y, (state["x"], state["w"]), state["dy"]))
    groups, w = sr.RowGroups(*state["plan"]), _blocks(sr, state["w"])
    if not case["train"]:
        return sr.adapter_linear(state["x"], w, state["down"], state["up"], groups,
                                 scale=state["scale"])
    y = sr.adapter_linear(state["x"], (w, _blocks(sr, state["w_t"])), state["down"],
                          state["up"], groups, scale=state["scale"], seed=_SEED)
    leaves = (state["x"], state["down"], state["up"])
    return (y.detach(), *torch.autograd.grad(y, leaves, state["dy"]))


def run(state):
    return _framework(state) if own else _PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------------------- exact --


def _exact_pow2(k):
    return ((k.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_held(x, name, draws=None):
    """FP64 values that a matrix's 1 x 128 blocks (or, with `draws` None and three
    dimensions, the 128 x 128 blocks of its last two) stand for."""
    square = x.dim() == 3
    x = x.double()
    rows, cols = x.shape[-2:]
    most, mantissa, low = _GRID[name]
    top = torch.nn.functional.pad(x.abs(), (0, -cols % _BLOCK, 0, -rows % _BLOCK if square else 0))
    top = top.unflatten(-1, (-1, _BLOCK)).amax(-1)
    if square:
        top = top.unflatten(-2, (-1, _BLOCK)).amax(-2).repeat_interleave(_BLOCK, -2)[..., :rows, :]
    top = top.repeat_interleave(_BLOCK, -1)[..., :cols]
    # the smallest power of two that brings the block's largest value onto the grid
    k = torch.ceil(torch.log2(top.clamp(min=2.0 ** -149) / most))
    k = torch.where(top > most * _exact_pow2(k), k + 1, k)
    k = torch.where(top <= most * _exact_pow2(k - 1), k - 1, k)
    k = torch.where(top == 0, torch.zeros_like(k), k.clamp(min=-127))
    y = x * _exact_pow2(-k)
    unit = _exact_pow2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** low))) - mantissa)
    steps = y.abs() / unit
    if draws is None:
        steps = torch.round(steps)
    else:
        steps = torch.trunc(steps) + (draws < torch.floor(torch.frac(steps) * 2.0 ** 24))
    return torch.sign(y) * steps * unit * _exact_pow2(k)


def _exact_draws(shape, copy, device):
    """Draws (24 bits) of a row-major matrix's elements for its stored copy 0 or 1."""
    key = _SEED ^ copy
    for shift, factor in ((16, 0x7FEB352D), (15, 0x846CA68B), (16, 1)):
        key = ((key ^ (key >> shift)) * factor) % 2 ** 32
    h = torch.remainder(torch.arange(shape[0] * shape[1], device=device) + key, 2 ** 32)
    for shift, factor in ((16, 0x7FEB352D), (15, 0x846CA68B), (16, 1)):
        h = torch.bitwise_xor(h, torch.div(h, 2 ** shift, rounding_mode="floor"))
        h = torch.remainder(h * factor, 2 ** 32)
    return torch.div(h, 256, rounding_mode="floor").reshape(shape)


def _exact_stored(data, scale):
    """FP64 values of kept blocks (128 x 128)."""
    rows, cols = data.shape[-2:]
    factor = _exact_pow2(scale.double() - 127).repeat_interleave(_BLOCK, -1)[..., :cols]
    return data.double() * factor.repeat_interleave(_BLOCK, -2)[..., :rows, :]


def _exact_expert(state):
    case, x = state["case"], state["x"].detach()
    held = _exact_held(x, "e4m3")
    ends = state["ends"].tolist()
    spans = [slice(a, b) for a, b in zip([0] + ends[:-1], ends)]
    tail = x.shape[0] - ends[-1]

    def behind(parts, cols):
        return torch.cat(parts + [torch.zeros((tail, cols), dtype=torch.float64,
                                              device=x.device)])

    if not case["train"]:
        return behind([held[s] @ _exact_stored(state["w"][0][e], state["w"][1][e]).mT
                       for e, s in enumerate(spans)], case["n"])
    dy, grad = state["dy"], case["grad"]
    by_row = _exact_held(dy, grad, _exact_draws(dy.shape, 0, x.device))
    draws = _exact_draws(dy.shape, 1, x.device)
    y, dx, dw = [], [], []
    for e, s in enumerate(spans):
        w = _exact_held(state["w"].detach()[e:e + 1], "e4m3")[0]
        y.append(held[s] @ w.mT)
        dx.append(by_row[s] @ w)
        dw.append(_exact_held(dy[s].mT, grad, draws[s].mT) @ _exact_held(x[s].mT, "e4m3").mT)
    return behind(y, case["n"]), behind(dx, case["k"]), torch.stack(dw)


def _exact_adapter(state):
    case, x = state["case"], state["x"].detach()
    index, x64 = state["index"], x.double()
    down, up = state["down"].detach().double(), state["up"].detach().double()
    scale = state["scale"].double()
    y = _exact_held(x, "e4m3") @ _exact_stored(*state["w"]).mT
    if case["train"]:
        dy = state["dy"].double()
        held = _exact_held(state["dy"], "e4m3", _exact_draws(dy.shape, 0, x.device))
        dx, ddown, dup = held @ _exact_stored(*state["w_t"]).mT, [], []
    for a in range(case["adapters"]):
        mine = scale[a] * (index == a).double()[:, None]
        if state["sizes"][a]:
            y += (mine * (x64 @ down[a].mT)) @ up[a].mT
        if case["train"]:
            g = mine * dy
            dx += (g @ up[a]) @ down[a]
            ddown.append((g @ up[a]).mT @ x64)
            dup.append(g.mT @ (x64 @ down[a].mT))
    return (y, dx, torch.stack(ddown), torch.stack(dup)) if case["train"] else y


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "group":
        order, ends = _plan(state["index"].tolist(), case["groups"])
        return _ints(order), _ints(ends)
    return _exact_expert(state) if case["op"] == "expert" else _exact_adapter(state)
