"""The experts' products outside the fused layer: what is measured, and their plain forms.

A program that trains or adapts a mixture-of-experts model, or serves one whose experts are bf16,
fp16 or int8, routes its tokens, brings the rows into expert order and multiplies each expert's
rows with that expert's matrix. How many rows an expert gets is known on the GPU (``counts``).

* ``grouped_mm``: the product in bf16 or fp16; in training with both gradients (``train``);
* ``int8_mm``: one matrix, int8 with a scale for each token and channel (a shared expert, a
  projection);
* ``grouped_int8_mm``: the same for each expert's rows;
* ``quantize``: rows to int8 with a scale for each row, before such a product.

Row counts run from one token to a training step's batch; the geometries are those of
``vibe_megakernel_amd.cases`` (hidden by intermediate, gate/up and down) and generic ones of odd
sizes.
"""

from __future__ import annotations

import functools
import hashlib
import importlib
import math

import torch

own = False

DEVICE = "cuda:0"

# experts, experts a token, hidden, intermediate, the most tokens drawn
GEOMETRIES = {
    "tiny": (8, 2, 1024, 512, 8192),
    "mixtral": (8, 2, 4096, 14336, 4096),
    "qwen3": (128, 8, 2048, 768, 8192),
    "glm": (288, 8, 4096, 2048, 512),
    "deepseek": (256, 8, 7168, 2048, 64),
}
TRAINED = ("tiny", "qwen3")  # geometries whose training step is drawn
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@functools.lru_cache(maxsize=None)  # a program imports the package once
def _products():
    import __graft_entry__

    __graft_entry__.load_package()  # the package directory's name is not an identifier
    return importlib.import_module("vibe_megakernel_amd.products")


def listed():
    return [
        # One user decoding on a small model: eight experts of one row each, so latency counts.
        dict(name="grouped-1tok", op="grouped_mm", E=128, tokens=1, topk=8, K=2048, N=768, dtype="bf16",
             transposed=False, tail=0, skew=0.0),
        # A decode batch on a large model: about 220 of 256 experts with a few rows each, so the weights stream.
        dict(name="grouped-decode64", op="grouped_mm", E=256, tokens=64, topk=8, K=7168, N=2048, dtype="bf16",
             transposed=False, tail=0, skew=0.0),
        # A prompt through few, wide experts: a thousand rows an expert, so the matrix cores decide.
        dict(name="grouped-prompt4096", op="grouped_mm", E=8, tokens=4096, topk=2, K=4096, N=14336, dtype="bf16",
             transposed=False, tail=0, skew=0.5),
        # Odd sizes, weights stored input-major, a buffer that is not full, experts of uneven load.
        dict(name="grouped-odd", op="grouped_mm", E=13, tokens=1237, topk=1, K=1000, N=1736, dtype="fp16",
             transposed=True, tail=211, skew=1.0),
        # A training step of a small model's experts: the product and both gradients.
        dict(name="train-32k", op="train", E=128, tokens=4096, topk=8, K=2048, N=768, dtype="bf16",
             transposed=False, tail=0, skew=0.5),
        # The gradients of a short adapter batch, a few experts unused.
        dict(name="train-short", op="train", E=8, tokens=75, topk=2, K=1024, N=512, dtype="fp16",
             transposed=False, tail=10, skew=2.0),
        # One token through a shared expert's projection.
        dict(name="int8-1tok", op="int8_mm", M=1, K=7168, N=2048, out="bf16"),
        # A prompt through a wide projection.
        dict(name="int8-prompt4096", op="int8_mm", M=4096, K=4096, N=14336, out="bf16"),
        # A decode batch on a large model with int8 experts.
        dict(name="grouped-int8-decode64", op="grouped_int8_mm", E=256, tokens=64, topk=8, K=7168, N=2048, out="bf16",
             tail=0, skew=0.0),
        # A prompt chunk's rows through many small int8 experts, an uneven load.
        dict(name="grouped-int8-2000", op="grouped_int8_mm", E=128, tokens=2000, topk=8, K=2048, N=768, out="bf16",
             tail=0, skew=1.0),
        # One token's activations to int8.
        dict(name="quantize-1tok", op="quantize", M=1, K=7168, dtype="bf16"),
        # A prompt's activations to int8.
        dict(name="quantize-prompt", op="quantize", M=16384, K=7168, dtype="bf16"),
    ]


def _spread(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.999))))))


def _odd_grouped(rng):
    """A generic geometry: any number of experts, sizes of no round multiple."""
    E = _spread(rng, 2, 64)
    step = rng.choice((1, 8, 8, 8))
    K, N = (step * _spread(rng, 64 // step, 2400 // step) for _ in range(2))
    return E, rng.randint(1, min(4, E)), K, N, 2048


def draw(rng):
    op = rng.choice(("grouped_mm", "grouped_mm", "train", "int8_mm", "grouped_int8_mm", "quantize"))
    if op == "quantize":
        K = rng.choice((_spread(rng, 64, 16384), 2048, 4096, 7168))
        return dict(op=op, M=_spread(rng, 1, min(65536, (16384 * 7168) // K)), K=K,
                    dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")))
    if op == "int8_mm":
        _, _, h, i, _ = GEOMETRIES[rng.choice(sorted(GEOMETRIES))]
        K, N = rng.choice(((h, i), (i, h), (_spread(rng, 64, 8192), _spread(rng, 64, 8192))))
        return dict(op=op, M=_spread(rng, 1, 4096), K=K, N=N, out=rng.choice(("bf16", "bf16", "fp16", "fp32")))
    if rng.random() < 0.4:
        E, topk, K, N, most = _odd_grouped(rng)
    else:
        E, topk, h, i, most = GEOMETRIES[rng.choice(TRAINED if op == "train" else sorted(GEOMETRIES))]
        K, N = rng.choice(((h, i), (i, h)))
    if op == "train":
        most = min(most, 4096)
    case = dict(op=op, E=E, tokens=_spread(rng, 1, most), topk=topk, K=K, N=N,
                tail=rng.choice((0, 0, rng.randint(1, 300))), skew=rng.choice((0.0, 0.5, 1.0, 2.0)))
    if op == "grouped_int8_mm":
        return dict(case, out=rng.choice(("bf16", "bf16", "fp16")))
    return dict(case, dtype=rng.choice(("bf16", "fp16")), transposed=rng.random() < 0.3)


def _generator(seed, name, device):
    digest = hashlib.blake2b(f"{seed}/{name}".encode(), digest_size=8).digest()
    return torch.Generator(device=device).manual_seed(int.from_bytes(digest, "little") & ((1 << 63) - 1))


def _normal(seed, name, shape, std, dtype):
    return torch.randn(shape, generator=_generator(seed, name, DEVICE), device=DEVICE, dtype=dtype).mul_(std)


def _int8(seed, name, shape):
    """Integers as a quantized normal variable gives them: the largest of a few thousand is near 127."""
    v = torch.randn(shape, generator=_generator(seed, name, DEVICE), device=DEVICE, dtype=torch.bfloat16)
    return v.mul_(36).round_().clamp_(-127, 127).to(torch.int8)


def _scales(seed, name, shape, about):
    return torch.rand(shape, generator=_generator(seed, name, DEVICE), device=DEVICE).add_(0.5).mul_(about)


def _counts(case, seed):
    """Rows an expert: every token picks its experts by a score with a bias for each expert."""
    g = _generator(seed, "routing", "cpu")
    noise = -torch.log(-torch.log(torch.rand((case["tokens"], case["E"]), generator=g).clamp_(1e-7, 1 - 1e-7)))
    bias = case["skew"] * torch.randn((1, case["E"]), generator=g)
    ids = (noise + bias).topk(case["topk"], dim=1).indices
    return torch.bincount(ids.flatten(), minlength=case["E"])


def _groups(case, seed):
    """The counts on the GPU, and the plan that a program without grouped products keeps for a
    padded batched product: the experts that have rows, each row's place, the longest group."""
    counts = _counts(case, seed)
    hit = counts.nonzero().flatten()
    c = counts[hit]
    start = torch.cumsum(c, 0) - c
    group = torch.repeat_interleave(torch.arange(len(hit)), c)
    place = torch.arange(int(c.sum())) - start[group]
    return {"counts": counts.to(DEVICE), "hit": hit.to(DEVICE), "group": group.to(DEVICE), "place": place.to(DEVICE),
            "longest": int(c.max()), "rows": int(c.sum())}


def prepare(case, seed):
    op = case["op"]
    state = {"op": op}
    if op == "quantize":
        # Activations: a normal body with a few channels that are far larger.
        x = _normal(seed, "x", (case["M"], case["K"]), 1.0, DTYPES[case["dtype"]])
        x[:, :: max(1, case["K"] // 6)] *= 20
        return dict(state, x=x)
    if op == "int8_mm":
        M, K, N = case["M"], case["K"], case["N"]
        return dict(state, x=_int8(seed, "x", (M, K)), xs=_scales(seed, "xs", (M,), 0.03),
                    w=_int8(seed, "w", (N, K)), ws=_scales(seed, "ws", (N,), 0.0006), out=DTYPES[case["out"]])
    state |= _groups(case, seed)
    E, K, N, R = case["E"], case["K"], case["N"], state["rows"] + case["tail"]
    if op == "grouped_int8_mm":
        return dict(state, x=_int8(seed, "x", (R, K)), xs=_scales(seed, "xs", (R,), 0.03),
                    w=_int8(seed, "w", (E, N, K)), ws=_scales(seed, "ws", (E, N), 0.0006), out=DTYPES[case["out"]])
    dtype = DTYPES[case["dtype"]]
    state |= {"x": _normal(seed, "x", (R, K), 1.0, dtype), "transposed": case["transposed"],
              "w": _normal(seed, "w", (E, K, N) if case["transposed"] else (E, N, K), 0.02, dtype)}
    if op == "train":
        state["dy"] = _normal(seed, "dy", (R, N), 0.01, dtype)
        state["x"].requires_grad_()
        state["w"].requires_grad_()
    return state


def _padded(rows, s):
    """[experts with rows, longest, ...] in 32 bits (64 for integers): the rows at their places, zeros elsewhere."""
    kind = torch.float64 if rows.dtype == torch.int8 else torch.float32
    out = torch.zeros((len(s["hit"]), s["longest"], rows.shape[1]), dtype=kind, device=rows.device)
    out[s["group"], s["place"]] = rows[: s["rows"]].to(kind)
    return out


def _unpadded(batch, s, rows):
    """The rows back in their order; rows of no expert are zero."""
    out = torch.zeros((rows, batch.shape[2]), dtype=batch.dtype, device=batch.device)
    out[: s["rows"]] = batch[s["group"], s["place"]]
    return out


def _plain_grouped(s):
    x, w = s["x"].detach(), s["w"].detach()
    hit = w[s["hit"]].float()
    right = hit if s["transposed"] else hit.transpose(1, 2).contiguous()
    xp = _padded(x, s)
    y = _unpadded(torch.bmm(xp, right), s, len(x)).to(x.dtype)
    if s["op"] == "grouped_mm":
        return y
    dy = _padded(s["dy"], s)
    dx = _unpadded(torch.bmm(dy, right.transpose(1, 2).contiguous()), s, len(x)).to(x.dtype)
    dw = torch.zeros_like(w)
    if s["transposed"]:
        dw[s["hit"]] = torch.bmm(xp.transpose(1, 2).contiguous(), dy).to(w.dtype)
    else:
        dw[s["hit"]] = torch.bmm(dy.transpose(1, 2).contiguous(), xp).to(w.dtype)
    return [y, dx, dw]


def _plain_quantize(x):
    v = x.float()
    largest = v.abs().amax(dim=1).clamp_min(2.0**-100)
    # (A number divided by a tensor is its reciprocal times the number: rounded twice.)
    q = torch.round(v * (torch.full_like(largest, 127.0) / largest)[:, None]).to(torch.int8)
    return [q, largest / 127.0]


def run(state):
    op = state["op"]
    if own:
        products = _products()
        if op == "quantize":
            return list(products.quantize_rows_int8(state["x"]))
        if op == "int8_mm":
            return products.int8_mm(state["x"], state["xs"], state["w"], state["ws"], out_dtype=state["out"])
        if op == "grouped_int8_mm":
            return products.grouped_int8_mm(state["x"], state["xs"], state["w"], state["ws"], state["counts"],
                                            out_dtype=state["out"])
        y = products.grouped_mm(state["x"], state["w"], state["counts"], transposed=state["transposed"])
        if op == "grouped_mm":
            return y
        return [y.detach(), *torch.autograd.grad(y, (state["x"], state["w"]), state["dy"])]
    if op == "quantize":
        return _plain_quantize(state["x"])
    # Integer sums pass 24 bits, so they are taken in 64.
    if op == "int8_mm":
        total = torch.mm(state["x"].double(), state["w"].double().t().contiguous())
        return (total * state["xs"][:, None] * state["ws"][None, :]).to(state["out"])
    if op == "grouped_int8_mm":
        x, xs, ws = state["x"], state["xs"], state["ws"][state["hit"]]
        right = state["w"][state["hit"]].double().transpose(1, 2).contiguous()
        total = torch.bmm(_padded(x, state), right) * ws[:, None, :]
        return (_unpadded(total, state, len(x)) * xs[:, None]).to(state["out"])
    return _plain_grouped(state)


def work(case):
    """Bytes and operations. The experts hit are counted as uniform routing would have them
    (1 - (1 - topk/E)^tokens of all); a skewed load hits no more."""
    op = case["op"]
    if op == "quantize":
        M, K = case["M"], case["K"]
        return {"bytes": M * K * (DTYPES[case["dtype"]].itemsize + 1) + 4 * M, "flops": 3 * M * K}
    K, N = case["K"], case["N"]
    if op == "int8_mm":
        M = case["M"]
        return {"bytes": M * K + N * K + 4 * (M + N) + M * N * DTYPES[case["out"]].itemsize, "flops": 2 * M * N * K}
    E, S = case["E"], case["tokens"] * case["topk"]
    R = S + case["tail"]
    hit = min(E, S, round(E * (1 - (1 - case["topk"] / E) ** case["tokens"])) if case["topk"] < E else E)
    hit = max(hit, case["topk"])
    if op == "grouped_int8_mm":
        return {"bytes": S * K + hit * N * K + 4 * (S + hit * N) + 8 * E + R * N * DTYPES[case["out"]].itemsize,
                "flops": 2 * S * N * K}
    if op == "grouped_mm":
        return {"bytes": 2 * (S * K + hit * N * K + R * N) + 8 * E, "flops": 2 * S * N * K}
    # x, dy and the weights read; y, dx and every expert's gradient written.
    return {"bytes": 2 * (S * K + S * N + hit * N * K + R * N + R * K + E * N * K) + 8 * E, "flops": 6 * S * N * K}


def exact(case, seed):
    """The definitions, expert by expert in 64 bits."""
    s = prepare(case, seed)
    op = s["op"]
    if op == "quantize":
        v = s["x"].double()
        largest = torch.maximum(v.max(dim=1).values, -v.min(dim=1).values).clamp_min(2.0**-100)
        return [None, largest / 127]
    if op == "int8_mm":
        return torch.einsum("mk,nk->mn", s["x"].double() * s["xs"].double()[:, None],
                            s["w"].double() * s["ws"].double()[:, None])
    rows, total = case["N"], len(s["x"])
    ends = torch.cumsum(s["counts"], 0).tolist()
    y = torch.zeros((total, rows), dtype=torch.float64, device=DEVICE)
    if op == "grouped_int8_mm":
        begin = 0
        for e, end in enumerate(ends):
            if end > begin:
                weight = s["w"][e].double() * s["ws"][e].double()[:, None]
                y[begin:end] = (s["x"][begin:end].double() * s["xs"][begin:end].double()[:, None]) @ weight.T
            begin = end
        return y
    x, w = s["x"].detach(), s["w"].detach()
    dx = torch.zeros((total, case["K"]), dtype=torch.float64, device=DEVICE)
    dw = torch.zeros(w.shape, dtype=torch.float64, device=DEVICE) if op == "train" else None
    begin = 0
    for e, end in enumerate(ends):
        if end > begin:
            matrix = w[e].double() if case["transposed"] else w[e].double().T
            xe = x[begin:end].double()
            y[begin:end] = xe @ matrix
            if op == "train":
                dye = s["dy"][begin:end].double()
                dx[begin:end] = dye @ matrix.T
                grad = xe.T @ dye
                dw[e] = grad if case["transposed"] else grad.T
        begin = end
    return y if op == "grouped_mm" else [y, dx, dw]
