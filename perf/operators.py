"""The packed 4-bit operators and the embedding, as measured: cases, inputs, one pass, exact values.

Two operators, each with its backward pass:

- ``int4_linear``: y = x W^T + b with a weight of 4-bit codes, W = (q - zp) * s with one scale and
  zero-point per group of input columns (or per row, or per tensor), and the gradients of x and b;
- ``embedding``: y[t] = scale * table[ids[t]] from a dense table or from a packed 4-bit one, and the
  gradient of a dense table, each row the sum over the tokens that looked it up.

``own`` chooses between the plain form (elementary torch operations in 32 bits, rounded once) and
the framework's calls.
"""

import functools
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _linear(name, tokens, n_in, n_out, dtype, group, sym, strategy="group", bias=False, train=False):
    return {"name": name, "op": "linear_train" if train else "linear", "tokens": tokens, "in": n_in, "out": n_out,
            "dtype": dtype, "strategy": strategy, "group": group, "sym": sym, "bias": bias}


def _embedding(name, tokens, vocab, hidden, dtype, scale, ids, packed=False, group=128, sym=True, padding=False,
               train=False):
    return {"name": name, "op": "embedding_train" if train else "embedding", "tokens": tokens, "vocab": vocab,
            "hidden": hidden, "dtype": dtype, "scale": scale, "ids": ids, "packed": packed, "group": group, "sym": sym,
            "padding": padding}


def listed():
    return [
        # One token through SmolLM2-135M's q_proj: the smallest call, all latency; 576 columns end
        # inside their fifth group of 128.
        _linear("decode_576x576_t1", 1, 576, 576, "bf16", 128, True),
        # One token through Llama-3-8B's down_proj, the W4A16 asymmetric g128 scheme GPTQ writes.
        _linear("decode_14336x4096_t1", 1, 14336, 4096, "bf16", 128, False),
        # Sixteen requests decoding together through Llama-3-8B's up_proj.
        _linear("decode_4096x14336_t16", 16, 4096, 14336, "fp16", 64, True),
        # SmolLM2-135M's tied output projection in fp32, one scale per vocabulary row.
        _linear("head_576x49152_t5_fp32", 5, 576, 49152, "fp32", 576, False, strategy="channel"),
        # A prompt of odd length through a layer of odd sizes with a bias.
        _linear("prompt_1000x1531_t333", 333, 1000, 1531, "fp16", 32, False, bias=True),
        # Four sequences of 2,048 tokens through Llama-3-8B's gate_proj: the largest product.
        _linear("prompt_4096x14336_t8192", 8192, 4096, 14336, "bf16", 128, False),
        # Adapter or norm tuning over frozen 4-bit weights: one sequence through Llama-3-8B's o_proj
        # and the gradient of its input.
        _linear("train_4096x4096_t2048", 2048, 4096, 4096, "bf16", 128, False, train=True),
        # The same in fp32 on SmolLM2-135M's up_proj, with a bias, a few short sequences.
        _linear("train_576x1536_t96_fp32", 96, 576, 1536, "fp32", 64, True, bias=True, train=True),
        # Decode step: the next tokens of seven requests from a packed 4-bit embedding table.
        _embedding("lookup_packed_49152x576_t7", 7, 49152, 576, "bf16", 1.0, "uniform", packed=True),
        # Calibration batch: 32 sequences of 2,048 tokens from a dense bf16 table, scaled by sqrt(hidden).
        _embedding("lookup_32000x4096_t65536", 65536, 32000, 4096, "bf16", 64.0, "zipf"),
        # SmolLM2-135M in fp32, the calibration set's 128 x 512 uniform tokens, with the table's gradient.
        _embedding("train_49152x576_t65536_fp32", 65536, 49152, 576, "fp32", 1.0, "uniform", train=True),
        # A training batch of Llama-3-8B's table: natural token frequencies and a padding token.
        _embedding("train_128256x4096_t16384", 16384, 128256, 4096, "bf16", 1.0, "zipf", padding=True, train=True),
    ]


LINEAR_MAX = 8192 * 4096 * 14336
TABLE_MAX = 128256 * 4096
TRAIN_MAX = 16384 * 4096


def _spread(rng, lo, hi):
    """A size between lo and hi, evenly over its logarithm; every second one a multiple of 64."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        n = max(64 if hi >= 64 and lo >= 32 else lo, n // 64 * 64 if n >= 64 else n)
    return min(max(n, lo), hi)


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if rng.random() < 0.6:
        train = rng.random() < 0.35
        n_in, n_out = _spread(rng, 64, 14336), _spread(rng, 64, 49152)
        most = LINEAR_MAX // (16 if dtype == "fp32" else 2 if train else 1) // (n_in * n_out)
        tokens = _spread(rng, 1, max(1, min(8192, most)))
        strategy = rng.choice(["group", "group", "group", "group", "channel", "tensor"])
        group = rng.choice([32, 64, 96, 128, 128, 256]) if strategy == "group" else n_in
        return _linear(None, tokens, n_in, n_out, dtype, group, rng.random() < 0.5, strategy, rng.random() < 0.3, train)
    train = rng.random() < 0.5
    vocab, hidden = _spread(rng, 64, 128256), _spread(rng, 64, 8192)
    while vocab * hidden * BYTES[dtype] > TABLE_MAX * 2:
        vocab = vocab // 2 + 1
    most = (TRAIN_MAX if train else 65536 * 4096) // hidden
    tokens = _spread(rng, 1, min(65536, most if dtype != "fp32" else most // 2))
    packed = not train and rng.random() < 0.5
    scale = rng.choice([1.0, math.sqrt(hidden), 0.5])
    return _embedding(None, tokens, vocab, hidden, dtype, scale, rng.choice(["uniform", "zipf"]), packed,
                      rng.choice([32, 64, 128]), rng.random() < 0.5, rng.random() < 0.4, train)


# ------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _codes(weight, strategy, group, sym):
    """4-bit codes of a weight as the framework's quantisers write them: (q - zp) & 0xF, two per byte
    with the even column in the high nibble, fp32 scales and int32 zero-points."""
    m, n = weight.shape
    if strategy == "tensor":
        low, high = weight.min().reshape(1, 1), weight.max().reshape(1, 1)
    elif strategy == "channel":
        low, high = weight.amin(1, keepdim=True), weight.amax(1, keepdim=True)
    else:
        groups = -(-n // group)
        padded = torch.cat([weight, weight[:, -1:].expand(m, groups * group - n)], 1).reshape(m, groups, group)
        low, high = padded.amin(2), padded.amax(2)
    if sym:
        scale = torch.maximum(low.abs(), high.abs()) / 7.0
        zero = torch.zeros_like(scale)
        least, most = -7, 7
    else:
        scale = (high - low) / 15.0
        zero = torch.round(-low / scale).clamp(0, 15)
        least, most = 0, 15
    columns = torch.arange(n, device=DEVICE) // group if strategy == "group" else torch.zeros(n, dtype=torch.long, device=DEVICE)
    q = torch.clamp(torch.round(weight / scale[:, columns]) + zero[:, columns], least, most)
    stored = (q - zero[:, columns]).to(torch.int32) & 0xF
    if n % 2:
        stored = torch.cat([stored, stored.new_zeros(m, 1)], 1)
    codes = (stored[:, 0::2] * 16 + stored[:, 1::2]).to(torch.uint8)
    shape = {"tensor": (1,), "channel": (m,)}.get(strategy, scale.shape)
    return {"codes": codes, "scales": scale.reshape(shape).contiguous(), "zero_points": zero.to(torch.int32).reshape(shape),
            "num_bits": 4, "symmetric": sym, "strategy": strategy, "group_size": group}


@functools.lru_cache(maxsize=8)
def _frequencies(vocab):
    """Token probabilities that fall off with the rank as in text."""
    p = 1.0 / (np.arange(vocab) + 2.7)
    return p / p.sum()


def _ids(case, g):
    vocab, tokens = case["vocab"], case["tokens"]
    if case["ids"] == "uniform":
        ids = torch.randint(0, vocab, (tokens,), generator=g, device=DEVICE)
    else:
        total = torch.from_numpy(np.cumsum(_frequencies(vocab))).to(DEVICE)
        u = torch.rand(tokens, generator=g, device=DEVICE, dtype=torch.float64)
        rank = torch.searchsorted(total, u).clamp(max=vocab - 1)
        ids = torch.randperm(vocab, generator=g, device=DEVICE)[rank]
    if case["padding"]:
        # The tail of each batch row is padding: an eighth of the positions hold token 0.
        ids = torch.where(torch.rand(tokens, generator=g, device=DEVICE) < 0.125, torch.zeros_like(ids), ids)
    return ids


def prepare(case, seed):
    g = _generator(seed)
    dtype = TYPES[case["dtype"]]
    state = {"case": case}
    if case["op"].startswith("linear"):
        m, n, t = case["out"], case["in"], case["tokens"]
        weight = torch.randn(m, n, generator=g, device=DEVICE) * 0.02
        entry = _codes(weight, case["strategy"], case["group"], case["sym"])
        x = torch.randn(t, n, generator=g, device=DEVICE)
        # A few channels of a transformer's activations are far larger than the rest.
        x = x * torch.where(torch.rand(n, generator=g, device=DEVICE) < 0.01, 20.0, 1.0)
        state["x"] = x.to(dtype)
        state["bias"] = torch.randn(m, generator=g, device=DEVICE).to(dtype) if case["bias"] else None
        if case["op"] == "linear_train":
            state["dy"] = (torch.randn(t, m, generator=g, device=DEVICE) * 0.01).to(dtype)
            if own:
                state["x"].requires_grad_(True)
                if case["bias"]:
                    state["bias"].requires_grad_(True)
    else:
        v, h, t = case["vocab"], case["hidden"], case["tokens"]
        table = torch.randn(v, h, generator=g, device=DEVICE) * 0.02
        entry = _codes(table, "group", case["group"], case["sym"]) if case["packed"] else None
        state["ids"] = _ids(case, g)
        if not case["packed"]:
            state["table"] = table.to(dtype)
        if case["op"] == "embedding_train":
            state["dy"] = (torch.randn(t, h, generator=g, device=DEVICE) * 0.01).to(dtype)
            if own:
                state["table"].requires_grad_(True)
    if entry is not None:
        state["entry"] = entry
        if own:
            import llmcompressorsharp_b200 as L

            state["weight"] = L.Int4Weight.from_entry(entry, case.get("in", case.get("hidden")))
    return state


# ------------------------------------------------------------------------------ one pass
def _dequantise(entry, n):
    """The fp32 weight (q - zp) * s of packed codes."""
    codes = entry["codes"].to(torch.int32)
    stored = torch.stack([codes >> 4, codes & 0xF], 2).reshape(codes.shape[0], -1)[:, :n]
    scale, zero = entry["scales"], entry["zero_points"]
    if entry["strategy"] == "group":
        columns = torch.arange(n, device=stored.device) // entry["group_size"]
        scale, zero = scale[:, columns], zero[:, columns]
    else:
        scale, zero = scale.reshape(-1, 1), zero.reshape(-1, 1)
    if entry["symmetric"]:
        value = torch.where(stored >= 8, stored - 16, stored)
    else:
        value = ((stored + zero) & 0xF) - zero
    return value.to(torch.float32) * scale


def _run_plain(state):
    case = state["case"]
    dtype = TYPES[case["dtype"]]
    if case["op"].startswith("linear"):
        weight = _dequantise(state["entry"], case["in"])
        y = state["x"].float() @ weight.t()
        if case["bias"]:
            y = y + state["bias"].float()
        out = [y.to(dtype)]
        if case["op"] == "linear_train":
            dy = state["dy"].float()
            out.append((dy @ weight).to(dtype))
            if case["bias"]:
                out.append(dy.sum(0).to(dtype))
        return out
    ids, scale = state["ids"], case["scale"]
    if case["packed"]:
        entry = state["entry"]
        rows = {k: (v[ids] if k in ("codes", "scales", "zero_points") else v) for k, v in entry.items()}
        return [(_dequantise(rows, case["hidden"]) * scale).to(dtype)]
    table = state["table"]
    out = [(table[ids].float() * scale).to(dtype)]
    if case["op"] == "embedding_train":
        grad = torch.zeros(table.shape, dtype=torch.float32, device=table.device)
        grad.index_add_(0, ids, state["dy"].float() * scale)
        if case["padding"]:
            grad[0] = 0
        out.append(grad.to(dtype))
    return out


def _run_own(state):
    import llmcompressorsharp_b200 as L

    case = state["case"]
    if case["op"].startswith("linear"):
        x, bias = state["x"], state["bias"]
        y = L.int4_linear(x, state["weight"], bias)
        if case["op"] == "linear":
            return [y]
        leaves = [x] + ([bias] if case["bias"] else [])
        return [y.detach(), *torch.autograd.grad(y, leaves, state["dy"])]
    padding = 0 if case["padding"] else None
    if case["packed"]:
        return [L.embedding(state["ids"], state["weight"], scale=case["scale"], padding_idx=padding, dtype=TYPES[case["dtype"]])]
    y = L.embedding(state["ids"], state["table"], scale=case["scale"], padding_idx=padding)
    if case["op"] == "embedding":
        return [y]
    return [y.detach(), *torch.autograd.grad(y, [state["table"]], state["dy"])]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------ work
def _distinct(case):
    """Expected number of different table rows that a batch looks up."""
    if case["ids"] == "uniform":
        p = np.full(case["vocab"], 1.0 / case["vocab"])
    else:
        p = _frequencies(case["vocab"])
    tokens = case["tokens"] * (0.875 if case["padding"] else 1.0)
    return float(np.sum(-np.expm1(tokens * np.log1p(-np.minimum(p, 1 - 1e-12)))))


def _packed_bytes(rows, n, strategy, group, sym):
    """Codes, an fp32 scale and (asymmetric) a byte of zero-point per group."""
    groups = {"tensor": 1, "channel": rows}.get(strategy, rows * -(-n // group))
    return rows * ((n + 1) // 2) + groups * (4 if sym else 5)


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"].startswith("linear"):
        t, n, m = case["tokens"], case["in"], case["out"]
        moved = _packed_bytes(m, n, case["strategy"], case["group"], case["sym"]) + e * t * (n + m) + (e * m if case["bias"] else 0)
        flops = 2 * t * n * m
        if case["op"] == "linear_train":
            moved += e * t * (n + m) + (e * m if case["bias"] else 0)
            flops *= 2
        return {"bytes": moved, "flops": flops}
    t, v, h = case["tokens"], case["vocab"], case["hidden"]
    rows = _distinct(case)
    table = _packed_bytes(rows, h, "group", case["group"], case["sym"]) if case["packed"] else rows * h * e
    moved = 8 * t + table + t * h * e
    flops = t * h
    if case["op"] == "embedding_train":
        moved += t * h * e + v * h * e
        flops += 2 * t * h
    return {"bytes": int(moved), "flops": flops}


# ------------------------------------------------------------------------------ exact values
def _integers(entry, n):
    """q - zp of packed codes in 64 bits, from the definition: the stored nibble is (q - zp) mod 16
    with q in [-7, 7] and zp = 0, or with q and zp in [0, 15]."""
    m = entry["codes"].shape[0]
    stored = torch.empty(m, 2 * entry["codes"].shape[1], dtype=torch.int64, device=DEVICE)
    stored[:, 0::2] = torch.div(entry["codes"], 16, rounding_mode="floor").to(torch.int64)
    stored[:, 1::2] = torch.remainder(entry["codes"], 16).to(torch.int64)
    stored = stored[:, :n]
    if entry["symmetric"]:
        return torch.remainder(stored + 8, 16) - 8
    zero = entry["zero_points"].to(torch.int64).reshape(m, -1) if entry["strategy"] != "tensor" else \
        entry["zero_points"].to(torch.int64).reshape(1, 1)
    if entry["strategy"] == "group":
        zero = zero.repeat_interleave(entry["group_size"], 1)[:, :n]
    return torch.remainder(stored + zero, 16) - zero


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"].startswith("linear"):
        n, entry = case["in"], state["entry"]
        values = _integers(entry, n).double()
        x = state["x"].detach().double()
        dy = state["dy"].double() if case["op"] == "linear_train" else None
        step = entry["group_size"] if entry["strategy"] == "group" else n
        y = torch.zeros(case["tokens"], case["out"], dtype=torch.float64, device=DEVICE)
        dx = torch.empty(x.shape, dtype=torch.float64, device=DEVICE) if dy is not None else None
        for first in range(0, n, step):
            part = slice(first, min(n, first + step))
            if entry["strategy"] == "group":
                scale = entry["scales"][:, first // step].double()
            else:
                scale = entry["scales"].double().reshape(-1).expand(case["out"])
            y += (x[:, part] @ values[:, part].t()) * scale
            if dy is not None:
                dx[:, part] = (dy * scale) @ values[:, part]
        if case["bias"]:
            y += state["bias"].detach().double()
        out = [y]
        if dy is not None:
            out.append(dx)
            if case["bias"]:
                out.append(torch.einsum("tm->m", dy))
        return out
    ids, scale = state["ids"], float(case["scale"])
    if case["packed"]:
        entry = state["entry"]
        rows = _integers(entry, case["hidden"])[ids].double()
        each = entry["scales"].double()[ids].repeat_interleave(entry["group_size"], 1)[:, : case["hidden"]]
        return [rows * each * scale]
    table = state["table"].detach()
    out = [table.double().index_select(0, ids).mul_(scale)]
    if case["op"] == "embedding_train":
        kept = ids != 0 if case["padding"] else torch.ones_like(ids, dtype=torch.bool)
        grad = torch.zeros(table.shape, dtype=torch.float64, device=DEVICE)
        grad.index_put_((ids[kept],), state["dy"][kept].double() * scale, accumulate=True)
        out.append(grad)
    return out
