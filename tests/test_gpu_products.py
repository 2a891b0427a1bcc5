"""``soap_tp_amd.products`` on the GPU against the formulas in 64 bits.

Tolerances, element by element.  A product's terms are exact in fp32 (16-bit operands) or rounded once
(fp32 operands); adding ``n`` of them in any order loses at most a step (2^-23, whichever way the adder
rounds) of the sum of magnitudes ``S`` per addition, so ``n * 2^-23 * S`` (one more for the rounded
terms of fp32); the result is rounded once to its type, by half a step of the value."""
import pytest
import torch

from soap_tp_amd import _native, products

pytestmark = pytest.mark.gpu

HALF = (torch.bfloat16, torch.float16)
TYPES = (*HALF, torch.float32)


def rounding(value, dtype):
    """Half a step of ``dtype`` at ``value`` (at least that of its smallest normal number's range)."""
    info = torch.finfo(dtype)
    return value.abs().clamp(min=info.tiny) * (info.eps / 2)


def assert_product(actual, expected, magnitudes, terms):
    """``expected`` and ``magnitudes`` (sums of the terms' magnitudes) in 64 bits."""
    summing = (terms + 1) * 2.0 ** -23 * magnitudes
    allowed = summing + rounding(expected.abs() + summing, actual.dtype)
    off = (actual.double() - expected).abs()
    assert actual.shape == expected.shape
    worst = (off - allowed).max().item() if off.numel() else 0.0
    assert worst <= 0, f"off by {off.max().item()} at most, {worst} over what rounding explains"


def split(tokens, experts, device, seed, spare=0):
    """Rows of each expert (some have none) and their ``ends``."""
    generator = torch.Generator().manual_seed(seed)
    cuts = torch.randint(0, tokens - spare + 1, (experts - 1,), generator=generator).sort().values.tolist()
    ends = [*cuts, tokens - spare]
    return list(zip([0, *ends[:-1]], ends)), torch.tensor(ends, dtype=torch.int64, device=device)


def values(device, seed, *shape, dtype):
    generator = torch.Generator(device=device).manual_seed(seed)
    return torch.randn(*shape, generator=generator, device=device).to(dtype)


def forward_exact(x, weights, spans):
    y = torch.zeros(x.shape[0], weights.shape[1], dtype=torch.float64, device=x.device)
    for e, (a, b) in enumerate(spans):
        y[a:b] = torch.mm(x[a:b].double(), weights[e].double().t())
    return y


def sums_exact(dy, x, spans):
    return torch.stack([torch.mm(dy[a:b].double().t(), x[a:b].double()) for a, b in spans])


def check_layer(device, dtype, tokens, experts, outputs, inputs, seed, spare=0, x=None, weights=None, dy=None):
    x = values(device, seed, tokens, inputs, dtype=dtype) if x is None else x
    weights = values(device, seed + 1, experts, outputs, inputs, dtype=dtype) if weights is None else weights
    dy = values(device, seed + 2, tokens, outputs, dtype=dtype) if dy is None else dy
    spans, ends = split(tokens, experts, device, seed, spare)
    y = products.expert_product(x, weights, ends)
    dx = products.expert_input_gradient(dy, weights, ends)
    dw = products.expert_weight_gradient(dy, x, ends)
    assert y.dtype == dx.dtype == dtype and dw.dtype == torch.float32
    turned = weights.transpose(1, 2)
    assert_product(y, forward_exact(x, weights, spans), forward_exact(x.abs(), weights.abs(), spans), inputs)
    assert_product(dx, forward_exact(dy, turned, spans), forward_exact(dy.abs(), turned.abs(), spans), outputs)
    assert_product(dw, sums_exact(dy, x, spans), sums_exact(dy.abs(), x.abs(), spans), max(1, tokens))
    rest = spans[-1][1]
    assert not y[rest:].any() and not dx[rest:].any()
    return x, weights, dy, spans, ends


# tokens, experts, outputs, inputs: from one token to several tiles, sizes on and off the tiles' edges and
# the 16-byte pieces, more experts than lanes of a wavefront, inner sizes of one and below a slab
SHAPES = [
    (1, 1, 8, 8), (1, 3, 16, 64), (2, 2, 1, 1), (16, 4, 32, 128), (17, 2, 33, 65), (33, 70, 40, 24), (100, 130, 24, 136),
    (127, 1, 128, 64), (128, 1, 127, 63), (129, 2, 136, 200), (300, 5, 72, 72), (257, 3, 130, 1), (64, 2, 1, 130),
    (500, 2, 264, 328), (1000, 4, 257, 129), (700, 1, 512, 1040),
    # long sums for few results: cut into parts
    (4100, 1, 136, 72), (5000, 2, 130, 257), (1100, 1, 8, 8),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_layer_products(device, shape, dtype):
    check_layer(device, dtype, *shape, seed=sum(shape))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_long_sums_with_and_without_a_workspace(device, dtype):
    """Through the C entry point: whole sums without a workspace, parts with one, and one that is too small."""
    tokens, outputs, inputs = 6000, 72, 80
    x, dy = values(device, 1, tokens, inputs, dtype=dtype), values(device, 2, tokens, outputs, dtype=dtype)
    need = _native.library().soapmi_expert_weight_gradient_workspace_bytes(1, tokens, outputs, inputs)
    assert need >= 2 * outputs * inputs * 4
    code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
    expected, magnitudes = sums_exact(dy, x, [(0, tokens)])[0], sums_exact(dy.abs(), x.abs(), [(0, tokens)])[0]

    def call(workspace, nbytes):
        dw = torch.empty(outputs, inputs, device=device)
        _native.call("soapmi_expert_weight_gradient", code, dy.data_ptr(), outputs, x.data_ptr(), inputs, None, 1, tokens,
                     outputs, inputs, 0, dw.data_ptr(), inputs, 0, workspace, nbytes,
                     torch.cuda.current_stream(device).cuda_stream)
        return dw

    work = torch.empty(need, dtype=torch.uint8, device=device)
    assert_product(call(None, 0), expected, magnitudes, tokens)
    assert_product(call(work.data_ptr(), need), expected, magnitudes, tokens)
    with pytest.raises(ValueError, match="workspace holds"):
        call(work.data_ptr(), need - 1)


@pytest.mark.parametrize("shape", [(1000, 4, 1024, 1100), (530, 3, 516, 1028), (700, 1, 1030, 1028), (259, 40, 260, 132)], ids=str)
def test_layer_products_in_single_precision(device, shape):
    """Sizes between a handful of rows and full tiles, rows at multiples of 16 bytes and not."""
    check_layer(device, torch.float32, *shape, seed=6, spare=5)


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("outputs,inputs", [(3600, 3584), (3601, 3590)], ids=str)
def test_layer_products_on_the_widest_tiles(device, dtype, outputs, inputs):
    check_layer(device, dtype, 3700, 2, outputs, inputs, seed=5, spare=60)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_rows_behind_the_last_expert(device, dtype):
    """New results have zeros there, a caller's buffer keeps what it had; NaN in such rows reaches nothing."""
    x, weights, dy, spans, ends = check_layer(device, dtype, 200, 3, 48, 56, seed=9, spare=37)
    calm = {48: products.expert_product(x, weights, ends), 56: products.expert_input_gradient(dy, weights, ends)}
    sums = products.expert_weight_gradient(dy, x, ends)
    x, dy = x.clone(), dy.clone()
    x[163:] = float("nan")
    dy[163:] = float("inf")
    for call, rows, width in ((products.expert_product, x, 48), (products.expert_input_gradient, dy, 56)):
        clean = calm[width][:163]
        fresh = call(rows, weights, ends)
        assert torch.equal(fresh[:163], clean) and not fresh[163:].any()
        out = torch.full((200, width), 7.0, dtype=dtype, device=device)
        assert call(rows, weights, ends, out=out) is out
        assert torch.equal(out[:163], clean) and (out[163:] == 7).all()
    assert torch.equal(products.expert_weight_gradient(dy, x, ends), sums)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_an_expert_sees_its_own_rows_only(device, dtype):
    """NaN and infinities in one expert's rows and weights stay with that expert."""
    spans, ends = [(0, 50), (50, 50), (50, 131), (131, 180)], torch.tensor([50, 50, 131, 180], device=device)
    x, dy = values(device, 1, 180, 40, dtype=dtype), values(device, 2, 180, 72, dtype=dtype)
    weights = values(device, 3, 4, 72, 40, dtype=dtype)
    clean = (products.expert_product(x, weights, ends), products.expert_input_gradient(dy, weights, ends),
             products.expert_weight_gradient(dy, x, ends))
    weights[1:3] = float("nan")
    x[50:131] = float("inf")
    dy[50:131] = float("nan")
    y, dx, dw = (products.expert_product(x, weights, ends), products.expert_input_gradient(dy, weights, ends),
                 products.expert_weight_gradient(dy, x, ends))
    for actual, expected in ((y, clean[0]), (dx, clean[1])):
        assert torch.equal(actual[:50], expected[:50]) and torch.equal(actual[131:], expected[131:])
        assert actual[50:131].isnan().all()
    assert torch.equal(dw[[0, 3]], clean[2][[0, 3]]) and not dw[1].any() and dw[2].isnan().all()


def strided(tensor, pad, offset):
    """The same values in rows that are ``pad`` elements longer and start ``offset`` elements in."""
    rows, columns = tensor.shape[-2:]
    store = torch.full((*tensor.shape[:-1], columns + pad + offset), 100, dtype=tensor.dtype, device=tensor.device)
    view = store[..., offset:offset + columns]
    view.copy_(tensor)
    return view


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("pad,offset", [(8, 0), (8, 8), (3, 0), (0, 1), (5, 2)])
def test_strides_and_alignment(device, dtype, pad, offset):
    x, weights, dy, spans, ends = check_layer(device, dtype, 150, 3, 136, 144, seed=21)
    views = [strided(t, pad, offset) for t in (x, weights, dy)]
    check_layer(device, dtype, 150, 3, 136, 144, seed=21, x=views[0], weights=views[1], dy=views[2])
    out = strided(torch.zeros(150, 136, dtype=dtype, device=device), pad, offset)
    products.expert_product(x, weights, ends, out=out)
    assert torch.equal(out, products.expert_product(x, weights, ends))
    dw = strided(torch.zeros(3, 136, 144, device=device), pad, offset)
    products.expert_weight_gradient(dy, x, ends, out=dw)
    assert torch.equal(dw, products.expert_weight_gradient(dy, x, ends))
    store = dw._base
    assert (store[..., :offset] == 100).all() and (store[..., offset + 144:] == 100).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(150, 3, 131, 141), (40, 2, 7, 9), (300, 1, 259, 66), (3700, 2, 3603, 75)], ids=str)
def test_aligned_rows_of_odd_length(device, shape, dtype):
    """Rows that start at multiples of 16 bytes and end anywhere: what stands between a row's end and the
    next one's start (here NaN) reaches nothing."""
    tokens, experts, outputs, inputs = shape

    def padded(seed, *size):
        store = torch.full((*size[:-1], -(-size[-1] // 8) * 8), float("nan"), dtype=dtype, device=device)
        store[..., :size[-1]] = values(device, seed, *size, dtype=dtype)
        return store[..., :size[-1]]

    x, weights, dy = padded(1, tokens, inputs), padded(2, experts, outputs, inputs), padded(3, tokens, outputs)
    check_layer(device, dtype, *shape, seed=sum(shape), x=x, weights=weights, dy=dy)


@pytest.mark.parametrize("tokens,outputs,inputs", [(40, 70, 141), (130, 200, 1090), (700, 260, 33), (3700, 3603, 75)])
def test_int8_product_of_aligned_rows_of_odd_length(device, tokens, outputs, inputs):
    generator = torch.Generator(device=device).manual_seed(inputs)
    pair = []
    for rows in (tokens, outputs):
        store = torch.randint(-128, 128, (rows, -(-inputs // 16) * 16), generator=generator, device=device, dtype=torch.int8)
        pair.append(store[:, :inputs])
    one = torch.ones(max(tokens, outputs), device=device)
    y = products.int8_product(pair[0], one[:tokens], pair[1], one[:outputs], out_dtype=torch.float32)
    assert torch.equal(y.double(), torch.mm(pair[0].double(), pair[1].double().t()))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_other_orders(device, dtype):
    """Column-major inputs, rows and experts that are the same memory."""
    x, weights, dy, spans, ends = check_layer(device, dtype, 90, 2, 40, 48, seed=33)
    check_layer(device, dtype, 90, 2, 40, 48, seed=33, x=x.t().contiguous().t(), dy=dy.t().contiguous().t(),
                weights=weights.transpose(1, 2).contiguous().transpose(1, 2))
    check_layer(device, dtype, 90, 2, 40, 48, seed=33, x=x[:1].expand(90, 48), weights=weights[:1].expand(2, 40, 48),
                dy=dy[:1, :1].expand(90, 40))


@pytest.mark.parametrize("dtype", HALF, ids=str)
def test_results_in_float32_and_in_the_inputs_type(device, dtype):
    x, weights, dy, spans, ends = check_layer(device, dtype, 150, 3, 72, 80, seed=41)
    wide = products.expert_product(x, weights, ends, out=torch.zeros(150, 72, device=device))
    assert_product(wide, forward_exact(x, weights, spans), forward_exact(x.abs(), weights.abs(), spans), 80)
    assert torch.equal(wide.to(dtype), products.expert_product(x, weights, ends))
    dw = products.expert_weight_gradient(dy, x, ends, out_dtype=dtype)
    assert dw.dtype == dtype and torch.equal(dw, products.expert_weight_gradient(dy, x, ends).to(dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("outputs", [3603, 3650, 3720])
def test_every_result_is_its_own_row_and_column(device, dtype, outputs):
    """Each result names its place: on the widest tiles, in both result types, with columns cut short."""
    tokens, inputs = 3840, 64
    x = torch.zeros(tokens, inputs, dtype=dtype, device=device)
    w = torch.zeros(outputs, inputs, dtype=dtype, device=device)
    rows, columns = torch.arange(tokens, device=device), torch.arange(outputs, device=device)
    x[:, 0], x[:, 1], x[:, 2] = (rows // 64).to(dtype), (rows % 64).to(dtype), 1
    w[:, 0], w[:, 1], w[:, 2], w[:, 3] = 64, 1, (columns % 128 / 128).to(dtype), 0
    expected = rows[:, None].double() + (columns % 128).double() / 128
    out = torch.zeros(tokens, outputs, device=device)
    assert torch.equal(products.expert_product(x, w, None, out=out).double(), expected)
    assert torch.equal(products.expert_product(x, w, None), out.to(dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_dense_layer(device, dtype):
    x, w, dy = values(device, 1, 70, 136, dtype=dtype), values(device, 2, 48, 136, dtype=dtype), values(device, 3, 70, 48, dtype=dtype)
    one = torch.tensor([70], device=device)
    assert torch.equal(products.expert_product(x, w, None), products.expert_product(x, w[None], one))
    assert torch.equal(products.expert_input_gradient(dy, w, None), products.expert_input_gradient(dy, w[None], one))
    assert torch.equal(products.expert_weight_gradient(dy, x, None), products.expert_weight_gradient(dy, x, one)[0])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_empty_extents(device, dtype):
    def empty(*shape):
        return torch.zeros(*shape, dtype=dtype, device=device)

    ends = torch.tensor([0, 0], device=device)
    assert products.expert_product(empty(0, 8), empty(2, 4, 8), ends).shape == (0, 4)
    dw = products.expert_weight_gradient(empty(0, 4), empty(0, 8), ends)
    assert dw.shape == (2, 4, 8) and not dw.any()
    ends = torch.tensor([2, 5], device=device)
    assert not products.expert_product(empty(5, 0), empty(2, 4, 0), ends).any()
    assert not products.expert_input_gradient(empty(5, 0), empty(2, 0, 8), ends).any()
    assert products.expert_product(empty(5, 8), empty(2, 0, 8), ends).shape == (5, 0)
    assert products.expert_weight_gradient(empty(5, 4), empty(5, 0), ends).shape == (2, 4, 0)
    none = torch.zeros(0, dtype=torch.int64, device=device)
    kept = torch.full((5, 4), 7.0, dtype=dtype, device=device)
    assert (products.expert_product(empty(5, 8) + 1, empty(0, 4, 8), none, out=kept) == 7).all()
    assert not products.expert_product(empty(5, 8) + 1, empty(0, 4, 8), none).any()
    assert products.expert_weight_gradient(empty(5, 4), empty(5, 8), none).shape == (0, 4, 8)


def test_ends_out_of_order_stay_inside_the_buffers(device):
    """Whatever ``ends`` holds, rows outside the buffers are neither read nor written."""
    for bad in ([300, -5, 90], [-(1 << 62), 1 << 62, 50], [1 << 40, 1 << 41, 1 << 42], [-3, -2, -1]):
        ends = torch.tensor(bad, device=device)
        x, weights = values(device, 1, 100, 64, dtype=torch.bfloat16), values(device, 2, 3, 32, 64, dtype=torch.bfloat16)
        dy = values(device, 3, 100, 32, dtype=torch.bfloat16)
        store = torch.full((300, 32), 7.0, dtype=torch.bfloat16, device=device)
        products.expert_product(x, weights, ends, out=store[100:200])
        assert (store[:100] == 7).all() and (store[200:] == 7).all()
        assert products.expert_weight_gradient(dy, x, ends).isfinite().all()
        assert products.expert_weight_gradient(dy, products.checkpoint_activations(x), ends).isfinite().all()


def check_part(actual, a, b):
    """Rows ``a`` times the matrix ``b``: other sizes may add in another order."""
    assert_product(actual, torch.mm(a.double(), b.double()), torch.mm(a.double().abs(), b.double().abs()), a.shape[1])


def test_offsets_beyond_32_bits(device):
    """Expert matrices and rows that start more than 2^32 bytes into their buffers."""
    inputs, outputs, experts = 4096, 8192, 72
    weights = torch.zeros(experts, outputs, inputs, dtype=torch.bfloat16, device=device)  # 4.5 GiB
    weights[-1] = values(device, 1, outputs, inputs, dtype=torch.bfloat16)
    x = values(device, 2, 40, inputs, dtype=torch.bfloat16)
    ends = torch.full((experts,), 20, dtype=torch.int64, device=device)
    ends[-1] = 40
    y = products.expert_product(x, weights, ends)
    assert not y[:20].any()
    check_part(y[20:], x[20:], weights[-1].t())
    dy = values(device, 3, 40, outputs, dtype=torch.bfloat16)
    dx = products.expert_input_gradient(dy, weights, ends)
    assert not dx[:20].any()
    check_part(dx[20:], dy[20:], weights[-1])
    products.expert_weight_gradient(dy, x, ends, out=weights)
    check_part(weights[-1], dy[20:].t(), x[20:])
    assert not weights[1:-1].any()
    del weights
    rows = 2200000  # of 1024 values in 16 bits: 4.5e9 bytes
    tall = torch.zeros(rows, 1024, dtype=torch.bfloat16, device=device)
    tall[-100:] = values(device, 4, 100, 1024, dtype=torch.bfloat16)
    small = values(device, 5, 16, 1024, dtype=torch.bfloat16)
    pair = torch.stack([small, small])
    ends = torch.tensor([rows - 100, rows], device=device)
    y = products.expert_product(tall, pair, ends)
    assert not y[:-100].any()
    check_part(y[-100:], tall[-100:], small.t())
    grown = products.expert_input_gradient(y, pair, ends)
    assert not grown[:-100].any()
    check_part(grown[-100:], y[-100:], small)
    dw = products.expert_weight_gradient(y, tall, ends)
    assert not dw[0].any()
    check_part(dw[1], y[-100:].t(), tall[-100:])
    saved = products.checkpoint_activations(tall)
    part = products.checkpoint_activations(tall[-100:])
    check_part(products.expert_weight_gradient(y, saved, ends)[1], y[-100:].t(), products.restore_activations(part))
    assert torch.equal(products.restore_activations(saved)[-100:], products.restore_activations(part))


# ---- activation checkpoints ----------------------------------------------------------------


def saved_exact(x):
    """The values a checkpoint of ``x`` stands for, from integer arithmetic on the bits of 64-bit floats."""
    wide = x.double()
    lowest = -24 if x.dtype == torch.float16 else -126
    kept = torch.empty_like(wide)
    for first in range(0, x.shape[1], 128):
        part = wide[:, first:first + 128]
        top = part.abs().amax(dim=1, keepdim=True)
        exponent = ((top.view(torch.int64) >> 52) - 1023 - 6).clamp(min=lowest)
        step = ((exponent + 1023) << 52).view(torch.float64)
        block = (part / step).round().clamp(-127, 127) * step
        kept[:, first:first + 128] = torch.where(top.isfinite(), block, torch.full_like(block, float("nan")))
    return kept


def awkward(device, dtype, rows, columns, seed):
    """Blocks of very different magnitudes: zeros, subnormal numbers, the type's largest, powers of two and
    values right at the edges between steps."""
    info = torch.finfo(dtype)
    x = values(device, seed, rows, columns, dtype=torch.float32)
    scale = 2.0 ** torch.randint(-12, 12, (rows, 1), generator=torch.Generator(device=device).manual_seed(seed), device=device)
    x = (x * scale).to(dtype)
    if rows >= 12:
        x[0] = 0
        x[1] = (x[1].float() * (info.smallest_normal / x[1].float().abs().max())).to(dtype)
        x[2] = info.max
        x[3] = -info.max
        x[3, ::3] = 1.0
        x[4] = 1.0
        x[5] = torch.arange(columns, device=device).to(dtype) / 2 - 30  # ties
        x[6] = torch.arange(columns, device=device).to(dtype) % 64 + 63.5
        x[7] = 0
        x[7, -1] = info.smallest_normal * info.eps
        x[8, 0] = float("nan")
        x[9, -1] = float("inf")
        x[10] = 127.75
    return x


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,columns", [(1, 1), (1, 4096), (12, 7), (13, 128), (40, 129), (33, 1000), (16, 4224)])
def test_checkpoint_and_restore(device, dtype, rows, columns):
    x = awkward(device, dtype, rows, columns, seed=rows + columns)
    saved = products.checkpoint_activations(x)
    assert saved.codes.shape == x.shape and saved.dtype == dtype
    assert saved.exponents.shape == (rows, -(-columns // 128))
    assert int(saved.codes.min()) >= -127
    restored = products.restore_activations(saved)
    expected = saved_exact(x)
    assert restored.dtype == dtype
    assert torch.equal(restored.isnan(), expected.isnan())
    assert torch.equal(restored.double().nan_to_num(), expected.nan_to_num())  # exactly
    finite = expected.isfinite()
    blocks = torch.nn.functional.pad(x.double().abs(), (0, -columns % 128)).view(rows, -1, 128).amax(dim=2)
    top = blocks.repeat_interleave(128, dim=1)[:, :columns]
    assert ((restored.double() - x.double()).abs() <= (top / 64).clamp(min=torch.finfo(dtype).tiny))[finite].all()
    view = strided(x, 3, 1)
    again = products.checkpoint_activations(view)
    assert torch.equal(again.codes, saved.codes) and torch.equal(again.exponents, saved.exponents)
    out = strided(torch.zeros_like(x), 3, 1)
    products.restore_activations(saved, out=out)
    assert torch.equal(out.nan_to_num(), restored.nan_to_num())
    plain = products.ActivationCheckpoint(saved.codes.contiguous(), saved.exponents, dtype)  # rows of any alignment
    assert torch.equal(products.restore_activations(plain).nan_to_num(), restored.nan_to_num())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1, 8, 8), (17, 2, 33, 65), (33, 70, 40, 24), (129, 2, 136, 200), (300, 5, 72, 328),
                                   (500, 2, 264, 520), (700, 1, 130, 1), (4100, 1, 136, 72), (5000, 2, 130, 257)], ids=str)
def test_weight_gradient_from_a_checkpoint(device, dtype, shape):
    tokens, experts, outputs, inputs = shape
    x = values(device, 1, tokens, inputs, dtype=dtype) * values(device, 2, 1, inputs, dtype=dtype)
    dy = values(device, 3, tokens, outputs, dtype=dtype)
    spans, ends = split(tokens, experts, device, seed=sum(shape), spare=tokens // 9)
    saved = products.checkpoint_activations(x)
    kept = saved_exact(x)
    expected, magnitudes = sums_exact(dy, kept, spans), sums_exact(dy.abs(), kept.abs(), spans)
    for checkpoint in (saved, saved._replace(codes=saved.codes.contiguous())):
        dw = products.expert_weight_gradient(dy, checkpoint, ends)
        assert_product(dw, expected, magnitudes, tokens)
    # a step that is a power of two enters exactly: the same product of the restored matrix has the same terms
    assert torch.equal(dw, products.expert_weight_gradient(dy, products.restore_activations(saved), ends))
    assert_product(products.expert_weight_gradient(strided(dy, 3, 1), saved, ends, out_dtype=dtype), expected, magnitudes, tokens)


@pytest.mark.parametrize("dtype", HALF, ids=str)
def test_weight_gradient_from_a_checkpoint_on_the_widest_tiles(device, dtype):
    x, dy = values(device, 1, 900, 3600, dtype=dtype), values(device, 2, 900, 3700, dtype=dtype)
    ends = torch.tensor([400, 880], device=device)
    saved = products.checkpoint_activations(x)
    spans, kept = [(0, 400), (400, 880)], saved_exact(x)
    assert_product(products.expert_weight_gradient(dy, saved, ends), sums_exact(dy, kept, spans),
                   sums_exact(dy.abs(), kept.abs(), spans), 480)


def test_weight_gradient_marks_columns_that_were_not_finite(device):
    x, dy = values(device, 1, 64, 384, dtype=torch.bfloat16), values(device, 2, 64, 32, dtype=torch.bfloat16)
    x[5, 200] = float("inf")
    dw = products.expert_weight_gradient(dy, products.checkpoint_activations(x), None)
    assert dw[:, 128:256].isnan().all() and dw[:, :128].isfinite().all() and dw[:, 256:].isfinite().all()


# ---- 8-bit integer product -----------------------------------------------------------------


def quantize_exact(x):
    wide = x.double()
    top = wide.abs().amax(dim=1, keepdim=True)
    codes = (127 * wide / torch.where(top > 0, top, torch.ones_like(top))).round()
    good = top.isfinite()
    scales = torch.where(good, top / 127, torch.full_like(top, float("nan")))
    return torch.where(good, codes, torch.zeros_like(codes)), scales[:, 0]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,columns", [(1, 1), (1, 4096), (12, 7), (13, 128), (40, 1000), (33, 1025), (16, 8200), (14, 9001)])
def test_quantize_tokens(device, dtype, rows, columns):
    x = awkward(device, dtype, rows, columns, seed=rows + columns)
    codes, scales = products.quantize_tokens(x)
    expected, steps = quantize_exact(x)
    # 127 x and the quotient are exact enough in fp32 for 16-bit values that no code differs; fp32 values
    # round 127 x, so that one next to the middle of two codes may go the other way
    exact = 127 * x.double() / x.double().abs().amax(dim=1, keepdim=True).clamp(min=1e-300)
    middle = (exact.abs() % 1 - 0.5).abs() <= (2.0 ** -15 if dtype == torch.float32 else 0)
    differ = codes.double() != expected
    if dtype == torch.float32:
        assert ((codes.double() - expected).abs() <= 1)[differ].all() and middle[differ].all()
    else:
        assert not differ.any()
    assert torch.equal(scales.isnan(), steps.isnan())
    allowed = (steps * 2.0 ** -24).clamp(min=2.0 ** -150)
    assert ((scales.double() - steps).abs() <= allowed)[steps.isfinite()].all()
    again = products.quantize_tokens(strided(x, 3, 1))
    assert torch.equal(again[0], codes) and torch.equal(again[1].nan_to_num(), scales.nan_to_num())


@pytest.mark.parametrize("out_dtype", TYPES, ids=str)
@pytest.mark.parametrize("tokens,outputs,inputs", [
    (1, 1, 1), (1, 4096, 1024), (2, 129, 16), (5, 33, 100), (16, 64, 128), (17, 130, 144), (70, 300, 272), (128, 128, 4096),
    (129, 257, 1000), (300, 1000, 1040), (40, 48, 0),
])
def test_int8_product(device, tokens, outputs, inputs, out_dtype):
    generator = torch.Generator(device=device).manual_seed(tokens + outputs + inputs)
    codes = torch.randint(-128, 128, (tokens, inputs), generator=generator, device=device, dtype=torch.int8)
    weights = torch.randint(-128, 128, (outputs, inputs), generator=generator, device=device, dtype=torch.int8)
    scales, channels = values(device, 1, tokens, dtype=torch.float32), values(device, 2, outputs, dtype=torch.float32)
    expected = torch.mm(codes.double(), weights.double().t()) * scales.double()[:, None] * channels.double()
    # the sum is rounded to fp32, then multiplied twice: three halves of a step
    allowed = expected.abs() * 3.01 * 2.0 ** -24
    allowed = allowed + rounding(expected.abs() + allowed, out_dtype)
    for a, b in ((codes, weights), (strided(codes, 3, 1), strided(weights, 16, 0))) if inputs else ((codes, weights),):
        y = products.int8_product(a, scales, b, channels, out_dtype=out_dtype)
        assert y.dtype == out_dtype and y.shape == expected.shape
        off = (y.double() - expected).abs()
        assert (off <= allowed)[expected.abs() < torch.finfo(out_dtype).max].all()


def test_int8_sums_are_exact_to_the_last_integer(device):
    """The largest sums there are, and the smallest difference from them."""
    inputs = 131071
    codes = torch.full((2, inputs), -128, dtype=torch.int8, device=device)
    weights = torch.full((3, inputs), -128, dtype=torch.int8, device=device)
    weights[1] = 127
    weights[2, ::2] = 127
    one = torch.ones(3, device=device)
    y = products.int8_product(codes, one[:2], weights, one, out_dtype=torch.float32)
    expected = torch.mm(codes.double(), weights.double().t()).float()
    assert torch.equal(y, expected)


def test_int8_product_on_the_widest_tiles(device):
    generator = torch.Generator(device=device).manual_seed(3)
    for tokens, outputs, inputs in ((3700, 3600, 528), (3700, 3590, 333)):
        codes = torch.randint(-127, 128, (tokens, inputs), generator=generator, device=device, dtype=torch.int8)
        weights = torch.randint(-127, 128, (outputs, inputs), generator=generator, device=device, dtype=torch.int8)
        y = products.int8_product(codes, torch.ones(tokens, device=device), weights, torch.ones(outputs, device=device),
                                  out_dtype=torch.float32)
        assert torch.equal(y.double(), torch.mm(codes.double(), weights.double().t()))


def test_a_token_that_was_not_finite_is_not_a_number(device):
    x, w = values(device, 1, 9, 64, dtype=torch.bfloat16), values(device, 2, 24, 64, dtype=torch.bfloat16)
    x[3, 5] = float("-inf")
    x[6] = 0
    y = products.int8_product(*products.quantize_tokens(x), *products.quantize_tokens(w))
    assert y[3].isnan().all() and not y[6].any() and y[[0, 1, 2, 4, 5, 7, 8]].isfinite().all()


# ---- as they are used ----------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("checkpoint", [False, True])
def test_expert_linear_gradients_are_the_formulas(device, dtype, checkpoint):
    x, weights = values(device, 1, 90, 136, dtype=dtype), values(device, 2, 3, 40, 136, dtype=dtype)
    spans, ends = [(0, 30), (30, 30), (30, 85)], torch.tensor([30, 30, 85], device=device)
    x.requires_grad_()
    weights.requires_grad_()
    y = products.expert_linear(x, weights, ends, checkpoint=checkpoint)
    dy = values(device, 3, 90, 40, dtype=dtype)
    y.backward(dy)
    kept = saved_exact(x.detach()) if checkpoint else x.detach()
    turned = weights.detach().transpose(1, 2)
    assert_product(y.detach(), forward_exact(x.detach(), weights.detach(), spans),
                   forward_exact(x.detach().abs(), weights.detach().abs(), spans), 136)
    assert_product(x.grad, forward_exact(dy, turned, spans), forward_exact(dy.abs(), turned.abs(), spans), 40)
    assert_product(weights.grad, sums_exact(dy, kept, spans), sums_exact(dy.abs(), kept.abs(), spans), 90)


def test_expert_linear_gradients_are_the_differences(device):
    """Along random directions: (f(p + h d) - f(p - h d)) / 2h of the quadratic f = sum((y - t)^2) / 2, which
    has no third derivative, so that the quotient is exact but for rounding: each f is off by at most
    ``terms * 2^-23`` of its sums of magnitudes (h = 1/4 keeps that small beside the difference)."""
    spans, ends = [(0, 20), (20, 33)], torch.tensor([20, 33], device=device)
    x, weights = values(device, 1, 33, 24, dtype=torch.float32), values(device, 2, 2, 16, 24, dtype=torch.float32)
    target = values(device, 3, 33, 16, dtype=torch.float32)

    def loss(x, w):
        return (products.expert_linear(x, w, ends) - target).double().square().sum() / 2

    xs, ws = x.clone().requires_grad_(), weights.clone().requires_grad_()
    loss(xs, ws).backward()
    resolved = []
    for seed in range(3):
        for base, grad, at in ((x, xs.grad, 0), (weights, ws.grad, 1)):
            d = values(device, 10 + seed, *base.shape, dtype=torch.float32)
            pair = []
            for sign in (0.25, -0.25):
                moved = [x, weights]
                moved[at] = base + sign * d
                pair.append(loss(*moved).item())
            quotient = (pair[0] - pair[1]) / 0.5
            slope = (grad.double() * d.double()).sum().item()
            magnitudes = forward_exact((x.abs() + d.abs() if at == 0 else x.abs()),
                                       (weights.abs() + d.abs() if at == 1 else weights.abs()), spans) + target.abs().double()
            allowed = 8 * (24 + 4) * 2.0 ** -23 * magnitudes.square().sum().item()
            assert abs(quotient - slope) <= allowed, (seed, at, quotient, slope, allowed)
            resolved.append(abs(slope) / allowed)
    assert max(resolved) > 20  # the bound says something


def test_expert_linear_frozen_parts(device):
    x, weights = values(device, 1, 30, 16, dtype=torch.bfloat16), values(device, 2, 2, 8, 16, dtype=torch.bfloat16)
    ends = torch.tensor([10, 30], device=device)
    frozen = products.expert_linear(x.clone().requires_grad_(), weights, ends, checkpoint=True)
    frozen.sum().backward()  # (a gradient whose elements are one value in memory)
    held = weights.clone().requires_grad_()
    products.expert_linear(x, held, ends, checkpoint=True).sum().backward()
    assert_product(held.grad, sums_exact(torch.ones(30, 8, device=device), saved_exact(x), [(0, 10), (10, 30)]),
                   sums_exact(torch.ones(30, 8, device=device), saved_exact(x).abs(), [(0, 10), (10, 30)]), 30)
    assert not products.expert_linear(x, weights, ends).requires_grad


@pytest.mark.parametrize("checkpoint", [False, True])
def test_a_layer_of_experts_trained_by_soap(device, checkpoint):
    """Forward, backward and the optimizer's step on every expert's gradient, as a training loop runs them:
    what soap_step is given is the weights' gradient, matrix by matrix, without a copy or a conversion."""
    from oracle import soap_oracle as oracle
    from soap_tp_amd import soap_step

    experts, outputs, inputs, tokens = 2, 24, 32, 64
    weights = values(device, 1, experts, outputs, inputs, dtype=torch.bfloat16)
    ends = torch.tensor([40, 64], device=device)
    spans = [(0, 40), (40, 64)]
    states, mirrors = [{} for _ in range(experts)], [{} for _ in range(experts)]
    config = dict(preconditioner_beta=0.9, beta1=0.9, beta2=0.95, eps=1e-6, basis_refresh_interval=100)
    for iteration in range(3):
        x = values(device, 100 + iteration, tokens, inputs, dtype=torch.bfloat16)
        held = weights.clone().requires_grad_()
        y = products.expert_linear(x, held, ends, checkpoint=checkpoint)
        dy = (y.detach().float() - values(device, 200 + iteration, tokens, outputs, dtype=torch.float32)).to(torch.bfloat16)
        y.backward(dy)
        kept = products.checkpoint_activations(x) if checkpoint else x
        dw = products.expert_weight_gradient(dy, kept, ends)
        assert torch.equal(dw.to(torch.bfloat16), held.grad)
        exact = sums_exact(dy, saved_exact(x) if checkpoint else x, spans)
        for e in range(experts):
            update = soap_step(dw[e], states[e], global_shape=(outputs, inputs), shard_dim=1, block_size=32,
                               process_grid_shape=(1, 1), **config)
            bases = {0: (states[e]["left_basis"].cpu().clone(), states[e]["right_basis"].cpu().clone())}
            expected = oracle.soap_step(exact[e].float().cpu(), mirrors[e], bases_override=bases, **config)
            error = (update.cpu().double() - expected.double()).norm() / max(expected.double().norm().item(), 1e-30)
            assert error <= 1e-4, (iteration, e, error)
            weights[e].add_(update, alpha=-0.01)


def test_a_served_layer_in_8_bits(device):
    """Weights quantised once, tokens one by one and as a prompt: the same rows either way."""
    w = values(device, 1, 200, 512, dtype=torch.bfloat16)
    x = values(device, 2, 40, 512, dtype=torch.bfloat16)
    plan = products.quantize_tokens(w)
    prompt = products.int8_product(*products.quantize_tokens(x), *plan)
    single = torch.cat([products.int8_product(*products.quantize_tokens(row[None]), *plan) for row in x])
    assert torch.equal(prompt, single)


# ---- streams, graphs, order ----------------------------------------------------------------


def _pass(x, weights, dy, ends, plan):
    saved = products.checkpoint_activations(x)
    return [products.expert_product(x, weights, ends), products.expert_input_gradient(dy, weights, ends),
            products.expert_weight_gradient(dy, x, ends), products.expert_weight_gradient(dy, saved, ends),
            products.restore_activations(saved), products.int8_product(*products.quantize_tokens(x), *plan)]


@pytest.mark.parametrize("dtype", HALF, ids=str)
def test_captured_and_replayed(device, dtype):
    """One graph, replayed with other inputs and other splits of the rows, eager work in between."""
    tokens, experts, outputs, inputs = 200, 3, 72, 264
    x, dy = (torch.empty(tokens, n, dtype=dtype, device=device) for n in (inputs, outputs))
    weights = torch.empty(experts, outputs, inputs, dtype=dtype, device=device)
    ends = torch.zeros(experts, dtype=torch.int64, device=device)
    plan = products.quantize_tokens(values(device, 9, outputs, inputs, dtype=dtype))

    def fill(seed):
        x.copy_(values(device, seed, tokens, inputs, dtype=dtype))
        dy.copy_(values(device, seed + 1, tokens, outputs, dtype=dtype))
        weights.copy_(values(device, seed + 2, experts, outputs, inputs, dtype=dtype))
        ends.copy_(split(tokens, experts, device, seed, spare=seed % 50)[1])

    fill(0)
    _pass(x, weights, dy, ends, plan)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = _pass(x, weights, dy, ends, plan)
    for seed in (10, 37, 60):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        for actual, expected in zip(captured, _pass(x, weights, dy, ends, plan)):
            assert torch.equal(actual, expected)


def test_long_sums_captured_and_replayed(device):
    """Sums cut into parts, with the parts' memory from the graph's own pool."""
    x, dy = (torch.empty(4000, n, dtype=torch.bfloat16, device=device) for n in (72, 136))

    def fill(seed):
        x.copy_(values(device, seed, 4000, 72, dtype=torch.bfloat16))
        dy.copy_(values(device, seed + 1, 4000, 136, dtype=torch.bfloat16))

    fill(0)
    products.expert_weight_gradient(dy, x, None)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = products.expert_weight_gradient(dy, x, None)
    for seed in (5, 9):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, products.expert_weight_gradient(dy, x, None))


def test_training_pass_captured_and_replayed(device):
    """Forward and backward pass through autograd in one graph, on other inputs and splits."""
    tokens, experts, outputs, inputs = 150, 4, 40, 136
    x, dy = (torch.zeros(tokens, n, dtype=torch.bfloat16, device=device) for n in (inputs, outputs))
    weights = torch.zeros(experts, outputs, inputs, dtype=torch.bfloat16, device=device)
    ends = torch.zeros(experts, dtype=torch.int64, device=device)
    leaves = x.requires_grad_(), weights.requires_grad_()

    def fill(seed):
        with torch.no_grad():
            x.copy_(values(device, seed, tokens, inputs, dtype=torch.bfloat16))
            dy.copy_(values(device, seed + 1, tokens, outputs, dtype=torch.bfloat16))
            weights.copy_(values(device, seed + 2, experts, outputs, inputs, dtype=torch.bfloat16))
            ends.copy_(split(tokens, experts, device, seed, spare=seed)[1])

    def eager():
        with torch.no_grad():
            saved = products.checkpoint_activations(x)
            return (products.expert_product(x, weights, ends), products.expert_input_gradient(dy, weights, ends),
                    products.expert_weight_gradient(dy, saved, ends, out_dtype=torch.bfloat16))

    fill(0)
    eager()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = products.expert_linear(x, weights, ends, checkpoint=True)
        captured = torch.autograd.grad(y, leaves, dy)
        y = y.detach()
    for seed in (3, 11, 20):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        for actual, expected in zip((y, *captured), eager()):
            assert torch.equal(actual, expected)


def test_columns_of_one_buffer(device):
    """A result written between the columns of its own input's buffer."""
    buffer = torch.zeros(50, 24, dtype=torch.bfloat16, device=device)
    buffer[:, :8] = values(device, 1, 50, 8, dtype=torch.bfloat16)
    w = values(device, 2, 16, 8, dtype=torch.bfloat16)
    expected = products.expert_product(buffer[:, :8].clone(), w, None)
    kept = buffer[:, :8].clone()
    products.expert_product(buffer[:, :8], w, None, out=buffer[:, 8:])
    assert torch.equal(buffer[:, 8:], expected) and torch.equal(buffer[:, :8], kept)


def test_two_streams_at_once_and_twice_the_same(device):
    x, weights = values(device, 1, 400, 256, dtype=torch.bfloat16), values(device, 2, 4, 192, 256, dtype=torch.bfloat16)
    dy = values(device, 3, 400, 192, dtype=torch.bfloat16)
    ends = torch.tensor([100, 100, 250, 390], device=device)
    plan = products.quantize_tokens(weights[0])
    expected = _pass(x, weights, dy, ends, plan)
    streams = [torch.cuda.Stream(device=device) for _ in range(2)]
    for stream in streams:
        stream.wait_stream(torch.cuda.current_stream(device))
    found = [[], []]
    for _ in range(4):
        for stream, into in zip(streams, found):
            with torch.cuda.stream(stream):
                into.append(_pass(x, weights, dy, ends, plan))
    torch.cuda.synchronize(device)
    for results in (*found[0], *found[1]):
        for actual, wanted in zip(results, expected):
            assert torch.equal(actual, wanted)


@pytest.mark.parametrize("dtype,inputs", [(torch.bfloat16, 8), (torch.bfloat16, 9), (torch.float32, 16)], ids=str)
def test_very_many_rows_of_short_products(device, dtype, inputs):
    """More tiles of few rows than a launch can have: a larger tile takes them."""
    tokens, outputs = 1 << 21, 4096
    x, w = values(device, 1, tokens, inputs, dtype=dtype), values(device, 2, outputs, inputs, dtype=dtype)
    y = products.expert_product(x, w, None)
    for first in range(0, tokens, 1 << 17):
        rows = slice(first, first + (1 << 17))
        wide = torch.mm(x[rows].double(), w.double().t())
        allowed = (inputs + 1) * 2.0 ** -23 * torch.mm(x[rows].double().abs(), w.double().abs().t())
        assert ((y[rows].double() - wide).abs() <= allowed + rounding(wide.abs() + allowed, dtype)).all()


@pytest.mark.parametrize("tokens", [3, 40, 3700])
@pytest.mark.parametrize("token,channel", [(1e34, 1e-6), (3e38, 1e-38), (-(2.0 ** 96), 2.0 ** -96), (1e-42, 1e30), (1e-45, 3e38),
                                           (1e30, 1e-40), (2.0 ** 127, 2.0 ** -149), (1e38, 1e20)])
def test_int8_scales_of_any_size(device, tokens, token, channel):
    """A token's scale alone may take the sum out of fp32's range, the channel's brings it back.  Roundings: the
    sum to fp32, two products, and what a subnormal result loses."""
    inputs, outputs = 64, 300
    generator = torch.Generator(device=device).manual_seed(tokens)
    codes = torch.randint(-127, 128, (tokens, inputs), generator=generator, device=device, dtype=torch.int8)
    weights = torch.randint(-127, 128, (outputs, inputs), generator=generator, device=device, dtype=torch.int8)
    codes[0], weights[0], weights[1] = 127, 127, 0  # the largest sum there is, and sums of zero
    scales, channels = torch.full((tokens,), token, device=device), torch.full((outputs,), channel, device=device)
    scales[-1] = 1.0
    expected = torch.mm(codes.double(), weights.double().t()) * scales.double()[:, None] * channels.double()
    y = products.int8_product(codes, scales, weights, channels, out_dtype=torch.float32).double()
    finite = expected.abs() <= torch.finfo(torch.float32).max * (1 - 4 * 2.0 ** -24)
    assert ((y - expected).abs() <= expected.abs() * 3.01 * 2.0 ** -24 + 2.0 ** -149)[finite].all()
    beyond = expected.abs() > torch.finfo(torch.float32).max * (1 + 4 * 2.0 ** -24)
    assert torch.equal(y[beyond], expected[beyond].sign() * float("inf"))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_restoring_every_exponent(device, dtype):
    """A checkpoint from elsewhere may hold any exponent; the values are codes * 2 ** (exponents - 127), rounded to the
    type (products of 2^-127 are subnormal in fp32 already, and exact there)."""
    codes = torch.arange(-127, 128, dtype=torch.int8, device=device).repeat(256, 1)
    exponents = torch.arange(256, device=device).to(torch.uint8)[:, None].repeat(1, 2)
    restored = products.restore_activations(products.ActivationCheckpoint(codes, exponents, dtype))
    steps = ((torch.arange(256, device=device) - 127 + 1023) << 52).view(torch.float64)
    expected = codes.double() * steps[:, None]
    expected[255] = float("nan")
    assert torch.equal(restored.nan_to_num(0.5), expected.to(dtype).nan_to_num(0.5))


@pytest.mark.parametrize("power", [-149 + 24, -60, 0, 127])
def test_codes_next_to_the_middle_of_two(device, power):
    """fp32 values right at the middles between codes and one step to each side: in 64 bits 127 x is exact, and a
    quotient of 31 by 24 bits that is not a middle is further from it than the rounding of 64 bits."""
    generator = torch.Generator(device=device).manual_seed(5)
    top = torch.rand(2000, 1, generator=generator, device=device) + 1
    top[0], top[1], top[2] = 1, 1.9921875, 127 / 64  # (the latter two are 127 / 64: middles that are fp32 values)
    middles = (torch.arange(-127, 127, device=device) + 0.5).double() * top.double() / 127
    x = middles.float()
    x = torch.cat([top, x, torch.nextafter(x, x + 1), torch.nextafter(x, x - 1), -top], dim=1)
    x = torch.ldexp(x, torch.tensor(power, device=device))
    codes, _ = products.quantize_tokens(x)
    expected = (127 * x.double() / x[:, :1].double()).round()
    assert torch.equal(codes.double(), expected)


def test_results_written_over_what_autograd_saved(device):
    """A saved tensor that a call overwrites is found in the backward pass, as with torch's own operations."""
    x, w = values(device, 1, 16, 32, dtype=torch.bfloat16), values(device, 2, 32, 32, dtype=torch.bfloat16)
    saved = products.checkpoint_activations(x)
    for rows, call in ((16, lambda out: products.expert_product(x, w, None, out=out)),
                       (16, lambda out: products.expert_input_gradient(x, w, None, out=out)),
                       (32, lambda out: products.expert_weight_gradient(x, w[:16], None, out=out)),
                       (16, lambda out: products.restore_activations(saved, out=out)),
                       (16, lambda out: products.int8_product(*products.quantize_tokens(x), *products.quantize_tokens(w), out=out))):
        kept = torch.zeros(rows, 32, dtype=torch.bfloat16, device=device)
        leaf = torch.ones_like(kept, requires_grad=True)
        product = leaf * kept
        call(kept)
        assert kept.any()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            product.sum().backward()
    held = torch.nn.Parameter(torch.zeros(16, 32, dtype=torch.bfloat16, device=device))
    with torch.no_grad():
        products.expert_product(x, w, None, out=held)
    assert torch.equal(held.detach(), products.expert_product(x, w, None))
    with torch.inference_mode():
        out = torch.zeros(16, 32, dtype=torch.bfloat16, device=device)
        products.expert_product(x, w, None, out=out)
    assert torch.equal(out, held.detach())


def test_expert_linear_keeps_what_its_gradients_need(device):
    """An operand may change before the backward pass if only its own gradient is asked for."""
    x, weights = values(device, 1, 30, 16, dtype=torch.bfloat16), values(device, 2, 2, 8, 16, dtype=torch.bfloat16)
    dy, ends = values(device, 3, 30, 8, dtype=torch.bfloat16), torch.tensor([10, 30], device=device)
    held = weights.clone().requires_grad_()
    y = products.expert_linear(x, held, ends)
    with torch.no_grad():
        held.mul_(2)  # (an optimizer's step)
    y.backward(dy)
    assert torch.equal(held.grad, products.expert_weight_gradient(dy, x, ends, out_dtype=torch.bfloat16))
    rows, frozen = x.clone().requires_grad_(), weights.clone()
    y = products.expert_linear(rows, frozen, ends)
    with torch.no_grad():
        rows.mul_(2)
    y.backward(dy)
    assert torch.equal(rows.grad, products.expert_input_gradient(dy, weights, ends))
    y = products.expert_linear(rows, frozen, ends)
    frozen.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy)


@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("x_dtype,weights_dtype", [(torch.float32, torch.float32), (None, torch.float32), (torch.float32, None),
                                                   (torch.bfloat16, torch.float16), (None, None)], ids=str)
def test_expert_linear_under_autocast(device, dtype, x_dtype, weights_dtype, checkpoint):
    """In autocast's type, whatever the operands' (None: that one); float32 weights get the sums' own float32."""
    x = values(device, 1, 90, 136, dtype=x_dtype or dtype).requires_grad_()
    weights = values(device, 2, 3, 40, 136, dtype=weights_dtype or dtype).requires_grad_()
    dy, ends = values(device, 3, 90, 40, dtype=dtype), torch.tensor([30, 30, 85], device=device)
    with torch.autocast("cuda", dtype=dtype):
        y = products.expert_linear(x, weights, ends, checkpoint=checkpoint)
    y.backward(dy)
    rows, matrices = x.detach().to(dtype), weights.detach().to(dtype)
    kept = products.checkpoint_activations(rows) if checkpoint else rows
    assert y.dtype == dtype and torch.equal(y.detach(), products.expert_product(rows, matrices, ends))
    assert torch.equal(x.grad, products.expert_input_gradient(dy, matrices, ends).to(x.dtype))
    sums = products.expert_weight_gradient(dy, kept, ends)
    assert torch.equal(weights.grad, sums if weights.dtype == torch.float32 else sums.to(dtype).to(weights.dtype))
    with torch.autocast("cuda", dtype=dtype), pytest.raises(ValueError, match="x must use float32, bfloat16 or float16"):
        products.expert_linear(x.double(), weights, ends)


def test_experts_trained_by_the_optimizer(device):
    """Experts' matrices as parameters of their own, in float32 under autocast: the optimizer takes each one's
    gradient as it is, and steps as soap_step does."""
    from soap_tp_amd import SOAP, soap_step

    experts, outputs, inputs, tokens = 3, 24, 32, 90
    ends = torch.tensor([40, 64, 85], device=device)
    weights = [torch.nn.Parameter(values(device, e, outputs, inputs, dtype=torch.float32)) for e in range(experts)]
    mirrors, states = [w.detach().clone() for w in weights], [{} for _ in weights]
    optimizer = SOAP(weights, lr=0.01, betas=(0.9, 0.95), eps=1e-6, weight_decay=0.0, precondition_frequency=100)
    for iteration in range(4):
        x = values(device, 100 + iteration, tokens, inputs, dtype=torch.bfloat16)
        dy = values(device, 200 + iteration, tokens, outputs, dtype=torch.bfloat16)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = products.expert_linear(x, torch.stack(weights), ends)
        y.backward(dy)
        dw = products.expert_weight_gradient(dy, x, ends)
        for e, w in enumerate(weights):
            assert torch.equal(w.grad, dw[e])
            update = soap_step(dw[e], states[e], global_shape=(outputs, inputs), shard_dim=1, block_size=128,
                               process_grid_shape=(1, 1), preconditioner_beta=0.95, beta1=0.9, beta2=0.95, eps=1e-6,
                               basis_refresh_interval=100)
            if iteration:
                mirrors[e] -= 0.01 * update
        optimizer.step()
        optimizer.zero_grad()
        for w, mirror in zip(weights, mirrors):
            assert (w.detach() - mirror).norm() <= 1e-5 * mirror.norm()


# ---- sums are held in 32 bits --------------------------------------------------------------
#
# The bound above grows with the terms, as a worst case does, and over thousands of them it would let sums in 16
# bits pass.  Whole numbers leave no room: every partial sum below 2^24 is exact in fp32, in any order, and odd
# ones above 2^11 are in neither of the 16-bit types.  For random values the norms are compared: a sum of n terms
# is rounded n times at most, each time by a step (2^-23) of a partial sum, which is sqrt(i / n) of the whole one
# after i terms; independent of each other, such errors have a root mean square below 2^-23 sqrt(n / 2) of the
# result's, and 8 times that is far below the 2^-9 sqrt(n / 2) and more of a sum kept in bf16 or the 2^-12 sqrt(n / 2)
# of one in fp16, even if it is rounded only every 64 rows.


def whole_numbers(device, seed, *shape, dtype):
    generator = torch.Generator(device=device).manual_seed(seed)
    return torch.randint(0, 9, shape, generator=generator, device=device).to(dtype)


LONG = [(6000, 1, 72, 80), (5000, 2, 130, 257), (4100, 3, 264, 3584), (3584, 1, 512, 4100), (40, 2, 16, 6000), (40, 2, 6000, 16)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", LONG, ids=str)
def test_long_sums_of_whole_numbers_are_exact(device, dtype, shape):
    tokens, experts, outputs, inputs = shape
    x, weights = whole_numbers(device, 1, tokens, inputs, dtype=dtype), whole_numbers(device, 2, experts, outputs, inputs, dtype=dtype)
    dy = whole_numbers(device, 3, tokens, outputs, dtype=dtype)
    spans, ends = split(tokens, experts, device, seed=sum(shape))
    wide = [torch.empty(tokens, n, device=device) for n in (outputs, inputs)]
    products.expert_product(x, weights, ends, out=wide[0])
    products.expert_input_gradient(dy, weights, ends, out=wide[1])
    assert torch.equal(wide[0].double(), forward_exact(x, weights, spans))
    assert torch.equal(wide[1].double(), forward_exact(dy, weights.transpose(1, 2), spans))
    expected = sums_exact(dy, x, spans)
    assert expected.max() < 2 ** 24 and (tokens < 1000 or (expected.max() > 2 ** 13 and (expected % 2 == 1).any()))
    assert torch.equal(products.expert_weight_gradient(dy, x, ends).double(), expected)
    assert torch.equal(products.expert_weight_gradient(dy, products.checkpoint_activations(x), ends).double(), expected)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", LONG, ids=str)
def test_long_sums_in_norm(device, dtype, shape):
    tokens, experts, outputs, inputs = shape
    x, weights = values(device, 1, tokens, inputs, dtype=dtype), values(device, 2, experts, outputs, inputs, dtype=dtype)
    dy = values(device, 3, tokens, outputs, dtype=dtype)
    spans, ends = split(tokens, experts, device, seed=sum(shape))

    def assert_near(actual, expected, terms):
        off, size = (actual.double() - expected).norm().item(), expected.norm().item()
        assert off <= 8 * 2.0 ** -23 * max(1.0, terms / 2) ** 0.5 * size, (off / size, terms)

    y, dx = torch.empty(tokens, outputs, device=device), torch.empty(tokens, inputs, device=device)
    products.expert_product(x, weights, ends, out=y)
    products.expert_input_gradient(dy, weights, ends, out=dx)
    assert_near(y, forward_exact(x, weights, spans), inputs)
    assert_near(dx, forward_exact(dy, weights.transpose(1, 2), spans), outputs)
    dw, expected = products.expert_weight_gradient(dy, x, ends), sums_exact(dy, x, spans)
    for e, (first, last) in enumerate(spans):  # with each expert's own number of terms, element by element too
        assert_near(dw[e], expected[e], last - first)
        magnitudes = torch.mm(dy[first:last].double().abs().t(), x[first:last].double().abs())
        assert_product(dw[e], expected[e], magnitudes, last - first)


def test_the_norms_would_show_sums_in_16_bits(device):
    """On the CPU: the same sizes with an accumulator that is rounded every 64 rows."""
    for tokens in (6000, 4100):
        x, dy = (values(torch.device("cpu"), seed, tokens, 64, dtype=torch.float32).bfloat16().float() for seed in (1, 2))
        expected = torch.mm(dy.double().t(), x.double())
        for kept in HALF:
            total = torch.zeros(64, 64)
            for first in range(0, tokens, 64):
                total = (total + torch.mm(dy[first:first + 64].t(), x[first:first + 64])).to(kept).float()
            assert (total.double() - expected).norm() > 8 * 2.0 ** -23 * (tokens / 2) ** 0.5 * expected.norm()


# ---- further from the ordinary -------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("stride_bytes", [(2 << 20) - 4096, 2 << 20, (8 << 20) - 4096, 8 << 20])
def test_rows_megabytes_apart(device, dtype, stride_bytes):
    """Around the distances beyond which rows are no longer fetched straight to LDS (2 MiB; for sums 8 MiB)."""
    stride = stride_bytes // torch.finfo(dtype).bits * 8
    tokens, outputs, inputs = 290, 130, 72

    def far(seed, rows, columns):
        view = torch.empty(rows * stride, dtype=dtype, device=device).as_strided((rows, columns), (stride, 1))
        return view.copy_(values(device, seed, rows, columns, dtype=dtype))

    x, dy = far(1, tokens, inputs), far(2, tokens, outputs)
    w = far(3, outputs, inputs)
    check_layer(device, dtype, tokens, 1, outputs, inputs, seed=4, x=x, dy=dy, weights=w[None])
    out = torch.empty(tokens * stride, dtype=dtype, device=device).as_strided((tokens, outputs), (stride, 1))
    assert torch.equal(products.expert_product(x, w, None, out=out), products.expert_product(x, w, None))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tokens,experts", [(3000, 5000), (40, 1000), (20000, 200)])
def test_many_experts(device, dtype, tokens, experts):
    check_layer(device, dtype, tokens, experts, 24, 40, seed=7, spare=3)


@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("tokens,experts,outputs,inputs", [(0, 2, 8, 16), (5, 0, 8, 16), (5, 2, 0, 16), (5, 2, 8, 0)])
def test_expert_linear_of_empty_extents(device, checkpoint, tokens, experts, outputs, inputs):
    x = torch.ones(tokens, inputs, device=device, requires_grad=True)
    weights = torch.ones(experts, outputs, inputs, device=device, requires_grad=True)
    ends = torch.full((experts,), tokens, dtype=torch.int64, device=device)
    y = products.expert_linear(x, weights, ends, checkpoint=checkpoint)
    assert y.shape == (tokens, outputs) and not y.any()
    y.backward(torch.ones_like(y))
    assert x.grad.shape == x.shape and not x.grad.any()
    assert weights.grad.shape == weights.shape and not weights.grad.any()


def test_calls_from_two_threads(device):
    """Each thread on a stream of its own, with other sizes, among them refused calls."""
    import threading

    def inputs(seed, tokens):
        return (values(device, seed, tokens, 256, dtype=torch.bfloat16), values(device, seed + 1, 4, 192, 256, dtype=torch.bfloat16),
                values(device, seed + 2, tokens, 192, dtype=torch.bfloat16), split(tokens, 4, device, seed)[1])

    def work(x, weights, dy, ends, plan, stream, into):
        with torch.cuda.device(device), torch.cuda.stream(stream):
            for _ in range(20):
                into.append(_pass(x, weights, dy, ends, plan))
                try:
                    products.expert_product(x, weights[:, :, :x.shape[0] % 200], ends)
                except ValueError as error:
                    into.append(str(error))

    cases, expected, found, threads = [], [], [], []
    for seed, tokens in ((1, 300), (20, 411)):
        case = inputs(seed, tokens)
        plan = products.quantize_tokens(case[1][0])
        cases.append((*case, plan))
        expected.append(_pass(*case, plan))
    torch.cuda.synchronize(device)
    for case in cases:
        found.append([])
        threads.append(threading.Thread(target=work, args=(*case, torch.cuda.Stream(device=device), found[-1])))
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    torch.cuda.synchronize(device)
    for case, results, wanted in zip(cases, found, expected):
        assert len(results) == 40
        message = f"x has 256 columns, expected {case[0].shape[0] % 200}."
        for result in results:
            if isinstance(result, str):
                assert result == message
            else:
                assert all(torch.equal(a, b) for a, b in zip(result, wanted))


def test_mixed_training_pass_captured_and_replayed(device):
    """Forward and backward pass under autocast in one graph: float32 weights, changed between the replays."""
    tokens, experts, outputs, inputs = 150, 4, 40, 136
    x, dy = torch.zeros(tokens, inputs, device=device), torch.zeros(tokens, outputs, dtype=torch.bfloat16, device=device)
    weights = torch.zeros(experts, outputs, inputs, device=device)
    ends = torch.zeros(experts, dtype=torch.int64, device=device)
    leaves = x.requires_grad_(), weights.requires_grad_()

    def fill(seed):
        with torch.no_grad():
            x.copy_(values(device, seed, tokens, inputs, dtype=torch.float32))
            dy.copy_(values(device, seed + 1, tokens, outputs, dtype=torch.bfloat16))
            weights.copy_(values(device, seed + 2, experts, outputs, inputs, dtype=torch.float32))
            ends.copy_(split(tokens, experts, device, seed, spare=seed)[1])

    def eager():
        with torch.no_grad():
            rows, matrices = x.bfloat16(), weights.bfloat16()
            saved = products.checkpoint_activations(rows)
            return (products.expert_product(rows, matrices, ends), products.expert_input_gradient(dy, matrices, ends).float(),
                    products.expert_weight_gradient(dy, saved, ends))

    fill(0)
    eager()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with torch.autocast("cuda", dtype=torch.bfloat16, cache_enabled=False):
            y = products.expert_linear(x, weights, ends, checkpoint=True)
        captured = torch.autograd.grad(y, leaves, dy)
        y = y.detach()
    for seed in (3, 11, 20):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        for actual, expected in zip((y, *captured), eager()):
            assert torch.equal(actual, expected)
