"""Cases of the matrix operators of low-precision training: Muon's orthogonalised
update, quantisation to 8-bit blocks and the products of such blocks.

Operators and the public calls they are reached through:

  orthogonalize   sr_states.orthogonalize(x)                  Newton-Schulz steps
  muon            sr_states.cuda.cuda_muon_step_(...)         momentum, orthogonalised update, parameter
  quantize        sr_states.quantize_blocks(x)                FP8 with a power-of-two scale a block of 128
  matmul          sr_states.matmul_blocks(a, b)               a @ b.T of two such tensors
  linear          sr_states.block_linear(x, weight)           a linear layer on them: forward and both
                                                              gradients (training), forward alone (serving)

``run`` computes the plain form with elementary torch operations in FP32, or
with ``own`` the framework's call.  ``exact`` computes the same outputs in FP64.
"""

import math
import sys

import torch

own = False

_PACKAGE = "stochastic-rounding-pytorch_b200"
_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
_EPS = 1e-7
_BLOCK = 128
_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16,
           "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
# Largest value, mantissa bits and exponent of the smallest normal number.
_GRID = {"e4m3": (448.0, 3, -6), "e5m2": (57344.0, 2, -14)}
_M32 = 0xFFFFFFFF


def _package():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    import sr_states
    import sr_states.cuda

    return sr_states


# ------------------------------------------------------------------- cases --

# Weight matrices of one GPT-2 small block and of one Llama-3-8B block (rows x columns).
_GPT2_BLOCK = "768x2304,768x768,768x3072,3072x768"
_LLAMA_BLOCK = "4096x4096,1024x4096,1024x4096,4096x4096,14336x4096,14336x4096,4096x14336"


def listed():
    return [
        # one small projection, the call a step of a toy model makes: launch latency counts
        {"name": "orth-1x128x512-f32", "op": "orthogonalize", "batch": 1, "m": 128, "n": 512,
         "dtype": "f32", "out": "bf16"},
        # the attention output projections of all GPT-2 small layers, stacked
        {"name": "orth-12x768x768-bf16", "op": "orthogonalize", "batch": 12, "m": 768, "n": 768,
         "dtype": "bf16", "out": "bf16"},
        # tall matrices of odd sizes (adapters, heads that no tile divides)
        {"name": "orth-3x1001x333-f32", "op": "orthogonalize", "batch": 3, "m": 1001, "n": 333,
         "dtype": "f32", "out": "bf16"},
        # a Llama-3-8B down projection, the largest matrix of its block
        {"name": "orth-1x4096x14336-bf16", "op": "orthogonalize", "batch": 1, "m": 4096,
         "n": 14336, "dtype": "bf16", "out": "bf16"},
        # the update of a GPT-2 small block: FP8 momentum, stochastically rounded
        {"name": "muon-gpt2-block-e4m3", "op": "muon", "shapes": _GPT2_BLOCK, "param": "bf16",
         "grad": "bf16", "state": "e4m3"},
        # the update of a Llama-3-8B block: BF16 momentum, stochastically rounded
        {"name": "muon-llama-block-bf16", "op": "muon", "shapes": _LLAMA_BLOCK, "param": "bf16",
         "grad": "bf16", "state": "bf16"},
        # the activations of a few decoded tokens
        {"name": "quant-8x4096-e4m3", "op": "quantize", "rows": 8, "cols": 4096, "src": "bf16",
         "dtype": "e4m3", "rounding": "nearest", "block": "row", "orientation": "rows"},
        # an output gradient on its way into both backward products
        {"name": "quant-8192x4096-both-e5m2-sr", "op": "quantize", "rows": 8192, "cols": 4096,
         "src": "bf16", "dtype": "e5m2", "rounding": "stochastic", "block": "row",
         "orientation": "both"},
        # one token through a Llama-3-8B up projection held in FP8: the weights' bytes bound it
        {"name": "linear-serve-1x4096x14336", "op": "linear", "tokens": 1, "k": 4096, "n": 14336,
         "train": False},
        # a prompt's product, the widest of Llama-3-8B
        {"name": "matmul-8192x14336x4096", "op": "matmul", "m": 8192, "n": 14336, "k": 4096,
         "a": "e4m3", "b": "e4m3", "b_block": "square", "out": "bf16"},
        # ragged product with sizes that no tile divides, E5M2 by E4M3
        {"name": "matmul-777x1000x1111", "op": "matmul", "m": 777, "n": 1000, "k": 1111,
         "a": "e5m2", "b": "e4m3", "b_block": "row", "out": "f32"},
        # a training step of a Llama-3-8B up projection: y, dx and dW
        {"name": "linear-train-4096x4096x14336", "op": "linear", "tokens": 4096, "k": 4096,
         "n": 14336, "train": True},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _odd(rng, size):
    """A size near `size`: half of the time a multiple of 128 or of 16, else as drawn."""
    step = rng.choice((1, 1, 16, 128))
    return max(step, size // step * step)


def draw(rng):
    op = rng.choice(("orthogonalize", "orthogonalize", "muon", "quantize", "matmul", "linear"))
    if op == "orthogonalize":
        m, n = _odd(rng, _log(rng, 64, 4096)), _odd(rng, _log(rng, 64, 14336))
        most = max(1, int(2e11 / (min(m, n) ** 2 * max(m, n))))
        return {"op": op, "batch": min(most, _log(rng, 1, 32)), "m": m, "n": n,
                "dtype": rng.choice(("f32", "bf16", "f16")), "out": rng.choice(("bf16", "f16"))}
    if op == "muon":
        kinds = [(_odd(rng, _log(rng, 64, 4096)), _odd(rng, _log(rng, 64, 4096)))
                 for _ in range(rng.randint(1, 3))]
        shapes = [rng.choice(kinds) for _ in range(rng.randint(1, 5))]
        return {"op": op, "shapes": ",".join("%dx%d" % s for s in shapes),
                "param": "bf16", "grad": rng.choice(("bf16", "f32")),
                "state": rng.choice(("f32", "bf16", "f16", "e4m3", "e5m2"))}
    if op == "quantize":
        return {"op": op, "rows": _odd(rng, _log(rng, 1, 8192)),
                "cols": _odd(rng, _log(rng, 64, 8192)), "src": rng.choice(("f32", "bf16", "f16")),
                "dtype": rng.choice(("e4m3", "e5m2")),
                "rounding": rng.choice(("nearest", "stochastic")),
                "block": rng.choice(("row", "row", "square")),
                "orientation": rng.choice(("rows", "columns", "both"))}
    if op == "matmul":
        return {"op": op, "m": _odd(rng, _log(rng, 1, 8192)), "n": _odd(rng, _log(rng, 64, 8192)),
                "k": _odd(rng, _log(rng, 64, 4096)), "a": rng.choice(("e4m3", "e5m2")),
                "b": rng.choice(("e4m3", "e5m2")), "b_block": rng.choice(("row", "square")),
                "out": rng.choice(("bf16", "f32", "f16"))}
    train = rng.random() < 0.5
    return {"op": op, "tokens": _log(rng, 64, 4096) if train else _log(rng, 1, 256),
            "k": _odd(rng, _log(rng, 128, 4096)), "n": _odd(rng, _log(rng, 128, 8192)),
            "train": train}


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


def _newton_flops(m, n, steps=5):
    # X X^T and its square are symmetric: half of each is enough
    m, n = min(m, n), max(m, n)
    return steps * (m * m * n + m * m * m + 2.0 * m * m * n)


def work(case):
    size = {k: torch.empty((), dtype=v).element_size() for k, v in _DTYPES.items()}
    op = case["op"]
    if op == "orthogonalize":
        count = case["batch"] * case["m"] * case["n"]
        return {"bytes": count * (size[case["dtype"]] + size[case["out"]]),
                "flops": case["batch"] * _newton_flops(case["m"], case["n"])}
    if op == "muon":
        each = 2 * size[case["param"]] + size[case["grad"]] + 2 * size[case["state"]]
        return {"bytes": sum(m * n for m, n in _shapes(case)) * each,
                "flops": sum(_newton_flops(m, n) for m, n in _shapes(case))}
    if op == "quantize":
        count = case["rows"] * case["cols"]
        copies = 2 if case["orientation"] == "both" else 1
        return {"bytes": count * (size[case["src"]] + copies), "flops": 0}
    if op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + m * n * size[case["out"]], "flops": 2.0 * m * n * k}
    t, k, n = case["tokens"], case["k"], case["n"]
    if not case["train"]:
        return {"bytes": n * k + 2 * t * (k + n), "flops": 2.0 * t * k * n}
    return {"bytes": 2 * (2 * t * k + 2 * t * n + 2 * n * k), "flops": 6.0 * t * k * n}


# ------------------------------------------------------------------ inputs --


def _matrix(gen, *shape):
    """A gradient-like matrix: noise, and as much energy in a few directions."""
    x = torch.randn(shape, generator=gen, device="cuda")
    left = torch.randn((*shape[:-1], 8), generator=gen, device="cuda")
    right = torch.randn((*shape[:-2], 8, shape[-1]), generator=gen, device="cuda")
    return x + 0.35 * (left @ right)


def _activations(gen, rows, cols):
    """Rows of different sizes and a few channels far above the rest, as activations have."""
    x = torch.randn((rows, cols), generator=gen, device="cuda")
    x *= torch.exp(0.5 * torch.randn((rows, 1), generator=gen, device="cuda"))
    x *= torch.exp(0.7 * torch.randn((1, cols), generator=gen, device="cuda"))
    return x


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    state = {"case": case, "seed": seed}
    if op == "orthogonalize":
        x = _matrix(gen, case["batch"], case["m"], case["n"]) * 1e-3
        state["x"] = x.to(_DTYPES[case["dtype"]])
    elif op == "muon":
        shapes = _shapes(case)
        state["param"] = [(torch.randn(s, generator=gen, device="cuda") * 0.02)
                          .to(_DTYPES[case["param"]]) for s in shapes]
        state["grad"] = [(_matrix(gen, *s) * 1e-2).to(_DTYPES[case["grad"]]) for s in shapes]
        state["momentum"] = [(_matrix(gen, *s) * 5e-2).to(_DTYPES[case["state"]]) for s in shapes]
    elif op == "quantize":
        state["x"] = _activations(gen, case["rows"], case["cols"]).to(_DTYPES[case["src"]])
    elif op == "matmul":
        a = _activations(gen, case["m"], case["k"])
        b = torch.randn((case["n"], case["k"]), generator=gen, device="cuda") * 0.02
        state["a"] = _quantize(a, case["a"], "nearest", "row", 0)
        state["b"] = _quantize(b, case["b"], "nearest", case["b_block"], 0)
    else:
        state["x"] = _activations(gen, case["tokens"], case["k"]).to(torch.bfloat16)
        w = (torch.randn((case["n"], case["k"]), generator=gen, device="cuda") * 0.02)
        if case["train"]:
            state["w"] = w.to(torch.bfloat16).requires_grad_()
            state["x"].requires_grad_()
            dy = _matrix(gen, case["tokens"], case["n"]) * 1e-4
            state["dy"] = dy.to(torch.bfloat16)
        else:
            # a server keeps its weights in FP8 with one scale a 128 x 128 block
            state["w"] = _quantize(w, "e4m3", "nearest", "square", 0)
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


def _hashes(shape, key, device):
    """The hash of every element of a row-major tensor: of its flat index plus `key`."""
    count = math.prod(shape)
    return _h32((torch.arange(count, device=device) + key) & _M32).view(shape)


def _pow2(k):
    """2^k in FP32 for whole k from -127 to 127, from its encoding."""
    k = k.to(torch.int32)
    return torch.where(k > -127, (k + 127) << 23, torch.full_like(k, 1 << 22)).view(torch.float32)


def _round(y, name, rounding, key):
    """FP32 `y` to the named type; 8-bit types saturate."""
    dtype = _DTYPES[name]
    if name == "f32":
        return y
    if name in _GRID:
        most, mantissa, low = _GRID[name]
        y = torch.where(torch.isnan(y), y, y.clamp(-most, most))
    else:
        mantissa, low = (7, -126) if name == "bf16" else (10, -14)
    if rounding == "nearest":
        return y.to(dtype)
    hashes = _hashes(y.shape, key, y.device)
    if name == "bf16":
        bits = (y.view(torch.int32).to(torch.int64) & _M32) + (hashes & 0xFFFF)
        bits = (bits >> 16) & 0xFFFF
        return torch.where(bits > 0x7FFF, bits - 0x10000, bits).to(torch.int16).view(dtype)
    exponent = (((y.view(torch.int32) >> 23) & 0xFF) - 127).clamp(min=low)
    unit = _pow2(exponent - mantissa)
    steps = y.abs() / unit
    whole = steps.floor()
    threshold = ((steps - whole) * 16777216.0).floor().to(torch.int64)
    up = ((hashes >> 8) < threshold).to(torch.float32)
    return torch.copysign((whole + up) * unit, y).to(dtype)


def _blocks(x, square):
    """`x` padded and viewed so that dimensions 1 and 3 run inside a block."""
    rows, cols = x.shape
    high = _BLOCK if square else 1
    x = torch.nn.functional.pad(x, (0, -cols % _BLOCK, 0, -rows % high))
    return x.view(x.shape[0] // high, high, x.shape[1] // _BLOCK, _BLOCK)


def _quantize(x, name, rounding, block, key, transposed=False):
    """(data, exponent + 127) of a tensor in blocks of 128 along its last dimension;
    `transposed`: of x.T, with the counters of x."""
    rows, cols = x.shape
    x = x.float()
    if transposed:
        x = x.t()
    square = block == "square"
    view = _blocks(x, square)
    size = torch.where(torch.isfinite(view), view.abs(), torch.zeros_like(view))
    top = size.amax(dim=(1, 3), keepdim=True)
    fraction, exponent = torch.frexp(top)  # top = fraction * 2^exponent, 0.5 <= fraction < 1
    ceiling = 9 if name == "e4m3" else 16  # the largest value is 0.875 * 2^ceiling
    k = exponent - ceiling + (fraction > 0.875).to(exponent.dtype)
    k = torch.where(top == 0, torch.zeros_like(k), k.clamp(min=-127))
    scaled = (view * _pow2(-k)).view(view.shape[0] * view.shape[1], -1)
    scaled = scaled[:x.shape[0], :x.shape[1]]
    if transposed:
        data = _round(scaled.t().contiguous(), name, rounding, key).t().contiguous()
    else:
        data = _round(scaled.contiguous(), name, rounding, key)
    return data, (k + 127).to(torch.uint8).view(k.shape[0], k.shape[2])


def _values(data, scale):
    """FP32 values of a quantised tensor."""
    rows, cols = data.shape
    factor = _pow2(scale.to(torch.int32) - 127).repeat_interleave(_BLOCK, 1)[:, :cols]
    if scale.shape[0] != rows:
        factor = factor.repeat_interleave(_BLOCK, 0)[:rows]
    return data.float() * factor


def _newton(x, steps=5):
    a, b, c = _COEFFICIENTS
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1)
    norm = x.square().sum(dim=(-2, -1), keepdim=True).sqrt()
    x = x / (norm + _EPS)
    for _ in range(steps):
        gram = x @ x.transpose(-2, -1)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(-2, -1) if tall else x


_LR, _MOMENTUM, _DECAY = 0.02, 0.95, 0.1


def _muon(state):
    case = state["case"]
    for i, (p, g, u) in enumerate(zip(state["param"], state["grad"], state["momentum"])):
        g32 = g.float()
        new = u.float() * _MOMENTUM + g32
        update = _newton(new * _MOMENTUM + g32)
        scale = max(1.0, p.shape[0] / p.shape[1]) ** 0.5
        p.copy_(p.float() * (1.0 - _LR * _DECAY) - (_LR * scale) * update)
        u.copy_(_round(new, case["state"], "stochastic", _key(1000 + i, 0)))
    return state["param"] + state["momentum"]


def _plain(state):
    case, op = state["case"], state["case"]["op"]
    if op == "orthogonalize":
        return _newton(state["x"].float()).to(_DTYPES[case["out"]]).contiguous()
    if op == "muon":
        return _muon(state)
    if op == "quantize":
        kinds = {"rows": (0,), "columns": (1,), "both": (0, 1)}[case["orientation"]]
        return [v for i in kinds for v in _quantize(state["x"], case["dtype"], case["rounding"],
                                                    case["block"], _key(5, i), bool(i))]
    if op == "matmul":
        return (_values(*state["a"]) @ _values(*state["b"]).t()).to(_DTYPES[case["out"]])
    x = _values(*_quantize(state["x"].detach(), "e4m3", "nearest", "row", 0))
    if not case["train"]:
        return (x @ _values(*state["w"]).t()).to(torch.bfloat16)
    w = _values(*_quantize(state["w"].detach(), "e4m3", "nearest", "square", 0))
    y = (x @ w.t()).to(torch.bfloat16)
    dy = state["dy"]
    rows = _values(*_quantize(dy, "e4m3", "stochastic", "row", _key(5, 0)))
    dx = (rows @ w).to(torch.bfloat16)
    columns = _values(*_quantize(dy, "e4m3", "stochastic", "row", _key(5, 1), True))
    tokens = _values(*_quantize(state["x"].detach(), "e4m3", "nearest", "row", 0, True))
    return y, dx, (columns @ tokens.t()).to(torch.bfloat16)


# --------------------------------------------------------------------- run --


def _framework(state):
    sr = _package()
    case, op = state["case"], state["case"]["op"]
    if op == "orthogonalize":
        return sr.orthogonalize(state["x"], dtype=_DTYPES[case["out"]])
    if op == "muon":
        sr.cuda.cuda_muon_step_(state["param"], state["grad"], state["momentum"], lr=_LR,
                                momentum_factor=_MOMENTUM, weight_decay=_DECAY,
                                seeds=[1000 + i for i in range(len(state["param"]))])
        return state["param"] + state["momentum"]
    if op == "quantize":
        got = sr.quantize_blocks(state["x"], dtype=_DTYPES[case["dtype"]],
                                 rounding=case["rounding"], seed=5,
                                 block=(_BLOCK, _BLOCK) if case["block"] == "square"
                                 else (1, _BLOCK), orientation=case["orientation"])
        both = got if case["orientation"] == "both" else (got,)
        return [v for t in both for v in (t.data, t.scale.view(torch.uint8))]
    if op == "matmul":
        a, b = (sr.BlockTensor(data, scale.view(torch.float8_e8m0fnu))
                for data, scale in (state["a"], state["b"]))
        return sr.matmul_blocks(a, b, dtype=_DTYPES[case["out"]])
    if not case["train"]:
        data, scale = state["w"]
        w = sr.BlockTensor(data, scale.view(torch.float8_e8m0fnu))
        return sr.block_linear(state["x"], w)
    y = sr.block_linear(state["x"], state["w"], seed=5)
    dx, dw = torch.autograd.grad(y, (state["x"], state["w"]), state["dy"])
    return y.detach(), dx, dw


def run(state):
    return _framework(state) if own else _plain(state)


# ------------------------------------------------------------------- exact --


def _exact_newton(x):
    """Newton-Schulz steps as one polynomial in the smaller Gram matrix at a time, in FP64."""
    c1, c3, c5 = _COEFFICIENTS
    x = x.double()
    x = x / (torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True) + _EPS)
    wide = x.shape[-1] >= x.shape[-2]
    eye = torch.eye(min(x.shape[-2:]), dtype=torch.float64, device=x.device)
    for _ in range(5):
        gram = x @ x.mT if wide else x.mT @ x
        factor = c1 * eye + gram @ (c3 * eye + c5 * gram)
        x = factor @ x if wide else x @ factor
    return x


def _exact_pow2(k):
    return ((k.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_scales(x, name, square):
    """Exponent of each block's power-of-two scale, by comparison with the grid's top."""
    top = torch.nan_to_num(x.double(), nan=0.0, posinf=0.0, neginf=0.0).abs()
    rows, cols = top.shape
    high = _BLOCK if square else 1
    top = torch.nn.functional.pad(top, (0, -cols % _BLOCK, 0, -rows % high))
    top = top.unflatten(1, (-1, _BLOCK)).amax(2).unflatten(0, (-1, high)).amax(1)
    k = torch.ceil(torch.log2(top.clamp(min=2.0 ** -149) / _GRID[name][0]))
    k = torch.where(top > _GRID[name][0] * _exact_pow2(k), k + 1, k)
    k = torch.where(top <= _GRID[name][0] * _exact_pow2(k - 1), k - 1, k)
    return torch.where(top == 0, torch.zeros_like(k), k.clamp(min=-127))


def _exact_spread(k, shape, square):
    k = k.repeat_interleave(_BLOCK, 1)[:, :shape[1]]
    return k.repeat_interleave(_BLOCK, 0)[:shape[0]] if square else k


def _exact_grid(y, name, draws=None):
    """FP64 `y` on an 8-bit grid: nearest, or up where the draw lies below the fraction."""
    most, mantissa, low = _GRID[name]
    y = y.clamp(-most, most)
    unit = _exact_pow2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** low))) - mantissa)
    steps = y.abs() / unit
    if draws is None:
        steps = torch.round(steps)
    else:
        part = torch.floor(torch.frac(steps) * 2.0 ** 24)
        steps = torch.trunc(steps) + (draws < part)
    return torch.sign(y) * steps * unit


def _exact_draws(shape, seed, index, transposed, device):
    rows, cols = (shape[1], shape[0]) if transposed else shape
    flat = torch.arange(rows * cols, device=device).reshape(rows, cols)
    flat = flat.t() if transposed else flat
    key = seed ^ index
    for shift, factor in ((16, 0x7FEB352D), (15, 0x846CA68B), (16, 1)):
        key = ((key ^ (key >> shift)) * factor) % 2 ** 32
    h = torch.remainder(flat + key, 2 ** 32)
    for shift, factor in ((16, 0x7FEB352D), (15, 0x846CA68B), (16, 1)):
        h = torch.bitwise_xor(h, torch.div(h, 2 ** shift, rounding_mode="floor"))
        h = torch.remainder(h * factor, 2 ** 32)
    return torch.div(h, 256, rounding_mode="floor")


def _exact_held(x, name, square, seed=None, index=0, transposed=False):
    """FP64 values that a tensor's blocks stand for."""
    x = x.double().t() if transposed else x.double()
    k = _exact_spread(_exact_scales(x, name, square), x.shape, square)
    draws = None if seed is None else _exact_draws(x.shape, seed, index, transposed, x.device)
    return _exact_grid(x * _exact_pow2(-k), name, draws) * _exact_pow2(k)


def _exact_stored(data, scale):
    k = scale.double() - 127
    return data.double() * _exact_pow2(_exact_spread(k, data.shape, k.shape[0] != data.shape[0]))


def exact(case, seed):
    state, op = prepare(case, seed), case["op"]
    if op == "orthogonalize":
        return _exact_newton(state["x"])
    if op == "muon":
        params, momenta = [], []
        for p, g, u in zip(state["param"], state["grad"], state["momentum"]):
            u = _MOMENTUM * u.double() + g.double()
            rows, cols = p.shape
            step = _LR * math.sqrt(max(1.0, rows / cols))
            params.append((1.0 - _LR * _DECAY) * p.double()
                          - step * _exact_newton(_MOMENTUM * u + g.double()))
            momenta.append(u)
        return params + momenta
    if op == "quantize":
        out, square = [], case["block"] == "square"
        for i in {"rows": (0,), "columns": (1,), "both": (0, 1)}[case["orientation"]]:
            x = state["x"].t() if i else state["x"]
            k = _exact_scales(x, case["dtype"], square)
            out += [x.double() * _exact_pow2(-_exact_spread(k, x.shape, square)),
                    (k + 127).to(torch.uint8)]
        return out
    if op == "matmul":
        return _exact_stored(*state["a"]) @ _exact_stored(*state["b"]).t()
    x = state["x"].detach()
    if not case["train"]:
        return _exact_held(x, "e4m3", False) @ _exact_stored(*state["w"]).t()
    w, dy = _exact_held(state["w"].detach(), "e4m3", True), state["dy"]
    y = _exact_held(x, "e4m3", False) @ w.t()
    dx = _exact_held(dy, "e4m3", False, 5, 0) @ w
    dw = (_exact_held(dy, "e4m3", False, 5, 1, True)
          @ _exact_held(x, "e4m3", False, None, 0, True).t())
    return y, dx, dw
