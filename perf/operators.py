"""The products of a layer whose weights SOAP trains, as cases that can be timed and checked.

Three operators.  Rows of ``x`` are tokens, sorted by expert; ``ends[e]`` is the first row behind expert ``e``'s
(a dense layer has no ``ends``: one expert holds every row); weights are (outputs, inputs) matrices.

* grouped products: ``y[t] = W[e(t)] x[t]``, and their gradients ``dx[t] = W[e(t)]^T dy[t]`` and
  ``dW[e] = sum over e's rows of dy[t] x[t]^T`` (the matrix that the optimizer takes);
* the product in 8-bit integers: rows of x and of W as codes in -127..127 with one scale for each row,
  ``y[t, n] = sx[t] sw[n] sum over k of qx[t, k] qw[n, k]``;
* activation checkpoints in 8 bits: codes in -127..127 with a power of two for each row and 128 columns, what they
  restore, and the weight gradient taken from them.

``own`` chooses between the plain form and the framework's calls.
"""
import numpy as np
import torch

own = False

BLOCK = 128  # columns that share an exponent in an activation checkpoint


# ---- cases ---------------------------------------------------------------------------------


def listed():
    return [
        # a decoding step of a mixture of experts: 32 (token, expert) rows, every expert's weights read once
        dict(name="expert_decode", op="product", dtype="bfloat16", tokens=32, spare=0, experts=8, out=3584, inp=4096, even=True),
        # the up projection of one training micro-batch, uneven routing and a padded buffer
        dict(name="expert_forward", op="product", dtype="bfloat16", tokens=4096, spare=128, experts=8, out=11008, inp=4096, even=False),
        # odd sizes in half precision: rows that start at no multiple of 16 bytes
        dict(name="expert_forward_odd", op="product", dtype="float16", tokens=1500, spare=3, experts=24, out=1111, inp=777, even=False),
        # both gradients of a small layer kept in single precision, as the optimizer's own matrices are
        dict(name="expert_backward_f32", op="backward", dtype="float32", tokens=1000, spare=0, experts=4, out=1024, inp=1100, even=False),
        # both gradients of a training micro-batch
        dict(name="expert_backward", op="backward", dtype="bfloat16", tokens=8192, spare=64, experts=8, out=2048, inp=4096, even=False),
        # a whole training pass through a wide layer: product, both gradients
        dict(name="expert_layer", op="layer", dtype="bfloat16", tokens=16384, spare=0, experts=16, out=3584, inp=4096, even=True),
        # one token of a served dense layer, its row quantised and multiplied
        dict(name="int8_single", op="int8", dtype="bfloat16", tokens=1, out=11008, inp=4096),
        # a short prompt through an odd-sized layer
        dict(name="int8_odd", op="int8", dtype="float16", tokens=333, out=1000, inp=1090),
        # a long prompt through a large layer
        dict(name="int8_prompt", op="int8", dtype="bfloat16", tokens=8192, out=14336, inp=4096),
        # saving a layer's activations and bringing them back
        dict(name="checkpoint_restore", op="restore", dtype="bfloat16", tokens=8192, inp=4096),
        # the weight gradient of a dense layer from activations saved in 8 bits
        dict(name="checkpoint_gradient", op="saved", dtype="bfloat16", tokens=8192, spare=0, experts=1, out=4096, inp=4096, even=True),
        # the same for experts with few rows each, odd sizes, half precision
        dict(name="checkpoint_gradient_odd", op="saved", dtype="float16", tokens=1023, spare=1, experts=5, out=520, inp=1000, even=False),
    ]


def draw(rng):
    def size(low, high, odd=0.3):
        value = int(round(np.exp(rng.uniform(np.log(low), np.log(high)))))
        return value if rng.random() < odd else max(16, value // 16 * 16)

    half = rng.choice(["bfloat16", "bfloat16", "float16"])
    op = rng.choice(["product", "backward", "layer", "int8", "restore", "saved"])
    if op == "restore":
        return dict(op=op, dtype=half, tokens=size(1, 8192, 1.0), inp=size(64, 8192))
    if op == "int8":
        return dict(op=op, dtype=half, tokens=size(1, 8192, 1.0), out=size(64, 11008), inp=size(64, 4096))
    dtype = "float32" if op != "saved" and rng.random() < 0.2 else half
    top = 1024 if dtype == "float32" else 4096
    experts = size(1, 32, 1.0)
    return dict(op=op, dtype=dtype, tokens=size(1, 2 * top, 1.0), spare=rng.choice([0, 0, 17]), experts=experts,
                out=size(64, top), inp=size(64, top), even=rng.random() < 0.5)


def prepare(case, seed):
    device = torch.device("cuda")
    dtype = getattr(torch, case["dtype"])
    generator = torch.Generator(device=device).manual_seed(seed)
    op, inp, tokens = case["op"], case["inp"], case["tokens"]
    rows = tokens + case.get("spare", 0)

    def normal(*shape):
        return torch.randn(*shape, generator=generator, device=device)

    # activations: some columns are far larger than the rest, and tokens differ in size
    width = torch.exp(0.7 * normal(inp)) * torch.exp(0.3 * normal(rows, 1))
    state = dict(case, x=(normal(rows, inp) * width).to(dtype))
    if op == "restore":
        return state
    if op == "int8":
        if rows > 8:
            state["x"][rows // 2] = 0  # a padding token
        codes, scales = _quantize(normal(case["out"], inp) * inp ** -0.5)
        state.update(weight_codes=codes, weight_scales=scales)
        return state
    experts = case["experts"]
    host = np.random.RandomState(seed % (1 << 32))
    share = host.dirichlet(np.full(experts, 50.0 if case["even"] else 1.0))
    counts = host.multinomial(tokens, share)
    ends = np.cumsum(counts)
    state["spans"] = [(int(end - count), int(end)) for end, count in zip(ends, counts)]
    state["ends"] = torch.from_numpy(ends.astype(np.int64)).to(device)
    if op != "saved":
        state["w"] = (normal(experts, case["out"], inp) * inp ** -0.5).to(dtype)
    if op != "product":
        state["dy"] = normal(rows, case["out"]).to(dtype)
    return state


# ---- plain forms ---------------------------------------------------------------------------


def _quantize(x):
    """Codes and scales of each row: scale = largest magnitude / 127, code = x / scale to the nearest even."""
    x = x.float()
    top = x.abs().amax(dim=1, keepdim=True)
    codes = torch.round(x * 127.0 / torch.where(top > 0, top, torch.ones_like(top)))
    return codes.to(torch.int8), (top / 127.0).squeeze(1)


def _save(x):
    """Codes and exponents of a checkpoint: with 2^(p-1) <= largest magnitude < 2^p the step is 2^(p-7)."""
    rows, columns = x.shape
    blocks = -(-columns // BLOCK)
    padded = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - columns)).view(rows, blocks, BLOCK)
    lowest = -24 if x.dtype == torch.float16 else -126
    exponents = (torch.frexp(padded.abs().amax(dim=2)).exponent - 7).clamp(min=lowest)
    steps = ((exponents + 127) << 23).view(torch.float32)  # 2^exponent, from its bits
    codes = torch.round(padded / steps[..., None]).clamp(-127, 127).to(torch.int8)
    return codes, steps


def _restore(codes, steps, columns):
    return (codes.float() * steps[..., None]).flatten(1)[:, :columns]


def _products(x, w, s):
    """Rows times their expert's matrix (w: experts x inner x columns); rows of no expert give zero."""
    parts = [x[a:b] @ w[e] for e, (a, b) in enumerate(s["spans"])]
    return torch.cat(parts + [x.new_zeros(x.shape[0] - s["spans"][-1][1], w.shape[2])])


def _gradients(dy, x, s):
    return torch.stack([dy[a:b].T @ x[a:b] for a, b in s["spans"]])


def run(s):
    op, x = s["op"], s["x"]
    dtype = x.dtype
    if own:
        from soap_tp_amd import products

        if op == "restore":
            return products.restore_activations(products.checkpoint_activations(x))
        if op == "int8":
            codes, scales = products.quantize_tokens(x)
            return products.int8_product(codes, scales, s["weight_codes"], s["weight_scales"], out_dtype=dtype)
        if op == "saved":
            return products.expert_weight_gradient(s["dy"], products.checkpoint_activations(x), s["ends"])
        out = {}
        if op != "backward":
            out["y"] = products.expert_product(x, s["w"], s["ends"])
        if op != "product":
            out["dx"] = products.expert_input_gradient(s["dy"], s["w"], s["ends"])
            out["dw"] = products.expert_weight_gradient(s["dy"], x, s["ends"])
        return out
    if op == "restore":
        return _restore(*_save(x), x.shape[1]).to(dtype)
    if op == "int8":
        codes, scales = _quantize(x)
        y = codes.float() @ s["weight_codes"].float().T
        return (y * scales[:, None] * s["weight_scales"]).to(dtype)
    if op == "saved":
        return _gradients(s["dy"].float(), _restore(*_save(x), x.shape[1]), s)
    out = {}
    if op != "backward":
        out["y"] = _products(x.float(), s["w"].float().transpose(1, 2), s).to(dtype)
    if op != "product":
        out["dx"] = _products(s["dy"].float(), s["w"].float(), s).to(dtype)
        out["dw"] = _gradients(s["dy"].float(), x.float(), s)
    return out


# ---- work and exact values -----------------------------------------------------------------


def work(case):
    op, tokens, inp = case["op"], case["tokens"], case["inp"]
    size = 4 if case["dtype"] == "float32" else 2
    if op == "restore":  # x in and out, codes written and read, an exponent for each block
        return dict(bytes=tokens * (inp * (2 * size + 2) + 2 * -(-inp // BLOCK)), flops=2 * tokens * inp)
    out = case["out"]
    product = 2 * tokens * out * inp
    if op == "int8":  # x read, codes and scales written and read, weight codes and scales read, y written
        return dict(bytes=tokens * (inp * (size + 2) + 8) + out * (inp + 4) + tokens * out * size, flops=product)
    weights = min(case["experts"], tokens) * out * inp  # of the experts that can have a row
    rows = tokens + case["spare"]
    if op == "product":
        return dict(bytes=size * (tokens * inp + weights + rows * out), flops=product)
    gradient = 4 * case["experts"] * out * inp
    if op == "saved":  # x read, codes written and read, dy read, dW written
        return dict(bytes=rows * (inp * (size + 1)) + tokens * (inp + out * size) + gradient, flops=product)
    backward = size * (tokens * (out + inp) + weights + rows * inp) + gradient
    forward = size * rows * out if op == "layer" else 0
    return dict(bytes=backward + forward, flops=(3 if op == "layer" else 2) * product)


def exact(case, seed):
    """The same values from the definitions, in 64 bits."""
    s = prepare(case, seed)
    op = case["op"]
    x = s["x"].double()
    if op == "int8":
        peak = x.abs().max(dim=1).values
        codes = torch.where(peak[:, None] > 0, (127 * x / peak[:, None]).round(), torch.zeros_like(x))
        return torch.einsum("tk,nk->tn", codes, s["weight_codes"].double()) * torch.outer(peak / 127, s["weight_scales"].double())
    if op in ("restore", "saved"):
        lowest = -24 if s["x"].dtype == torch.float16 else -126
        kept = torch.empty_like(x)
        for first in range(0, x.shape[1], BLOCK):
            part = x[:, first:first + BLOCK]
            peak = part.abs().max(dim=1, keepdim=True).values
            power = (peak.view(torch.int64) >> 52) - 1023 - 6  # from the bits: log2 and pow may round
            step = ((power.clamp(min=lowest) + 1023) << 52).view(torch.float64)
            kept[:, first:first + BLOCK] = (part / step).round().clamp(-127, 127) * step
        x = kept
        if op == "restore":
            return x
    expert = torch.bucketize(torch.arange(x.shape[0], device=x.device), s["ends"], right=True)
    found = {}
    if op != "saved":
        w = s["w"].double()
        found["y"] = x.new_zeros(x.shape[0], case["out"])
        found["dx"] = torch.zeros_like(x)
    found["dw"] = x.new_zeros(case["experts"], case["out"], case["inp"])
    for e in range(case["experts"]):
        mine = torch.nonzero(expert == e).flatten()
        if op in ("product", "layer"):
            found["y"][mine] = torch.mm(x[mine], w[e].t())
        if op != "product":
            dy = s["dy"][mine].double()
            found["dw"][e] = torch.mm(dy.t(), x[mine])
            if op != "saved":
                found["dx"][mine] = torch.mm(dy, w[e])
    if op == "saved":
        return found["dw"]
    return {"product": {"y": found["y"]}, "backward": {"dx": found["dx"], "dw": found["dw"]}, "layer": found}[op]
