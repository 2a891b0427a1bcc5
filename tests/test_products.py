"""Host-side checks of ``soap_tp_amd.products`` that need no GPU: every refusal is raised before
anything is launched, by the Python layer and by the C entry points."""
import pytest
import torch

import soap_tp_amd
from soap_tp_amd import _native, build, products

P = 4096  # a non-null address that no refused call dereferences


def _ends(*values):
    return torch.tensor(values, dtype=torch.int64)


def test_products_are_public():
    assert soap_tp_amd.products is products
    assert sorted(products.__all__) == [
        "ActivationCheckpoint", "checkpoint_activations", "expert_input_gradient", "expert_linear", "expert_product",
        "expert_weight_gradient", "int8_product", "quantize_tokens", "restore_activations"]
    for name in products.__all__:
        assert getattr(products, name).__doc__


X, W, DY = torch.zeros(6, 8), torch.zeros(2, 4, 8), torch.zeros(6, 4)


@pytest.mark.parametrize("arguments,message", [
    (dict(x=torch.zeros(8)), "x must be 2D"),
    (dict(x=[1.0]), "x must be a tensor"),
    (dict(x=X.double()), "x must use float32, bfloat16 or float16"),
    (dict(weights=torch.zeros(4, 8)), "weights must be 3D"),
    (dict(ends=None), "weights must be 2D"),
    (dict(weights=W.half()), "weights must use torch.float32"),
    (dict(x=torch.zeros(6, 7)), "x has 7 columns, expected 8"),
    (dict(ends=_ends(1, 2, 3)), "ends has 3 entries"),
    (dict(ends=_ends(3, 6).int()), "ends must use int64"),
    (dict(ends=_ends(3, 0, 6, 0)[::2]), "ends must be contiguous"),
    (dict(ends=_ends(3, 6).view(1, 2)), "ends must be 1D"),
    (dict(out=torch.zeros(6, 5)), "out has shape"),
    (dict(out=torch.zeros(6, 4).half()), "out must use torch.float32"),
    (dict(out=torch.zeros(4, 6).T), "out must have contiguous rows"),
    (dict(out=torch.zeros(1, 4).expand(6, 4)), "out must have contiguous rows"),
    (dict(out=X[:, 1:5]), "out must not overlap x"),
    (dict(out=W.view(-1)[:24].view(6, 4)), "out must not overlap weights"),
    (dict(), "requires cuda buffers"),
])
def test_expert_product_refusals(arguments, message):
    call = dict(x=X, weights=W, ends=_ends(3, 6), **{"out": None})
    call.update(arguments)
    with pytest.raises(ValueError, match=message):
        products.expert_product(call["x"], call["weights"], call["ends"], out=call["out"])


def test_overlap_is_that_of_elements():
    """Different columns of one buffer are apart, however their memory interleaves."""
    buffer = torch.zeros(6, 20)
    a, b = buffer[:, :8], buffer[:, 8:20]
    assert products._apart(a, b) and products._apart(b, a)
    assert not products._apart(buffer[:, :9], b) and not products._apart(b, buffer[:, 4:9])
    assert products._apart(buffer[:3], buffer[3:]) and not products._apart(buffer[:4], buffer[3:])
    assert not products._apart(a, buffer.view(12, 10)[:, 8:])  # other strides that meet
    assert not products._apart(buffer.t(), b)
    with pytest.raises(ValueError, match="requires cuda buffers"):  # not "overlap"
        products.expert_product(buffer[:, :8], torch.zeros(12, 8), None, out=buffer[:, 8:])


def test_input_gradient_refusals():
    with pytest.raises(ValueError, match="gradient has 8 columns, expected 4"):
        products.expert_input_gradient(X, W, _ends(3, 6))
    with pytest.raises(ValueError, match="requires cuda buffers"):
        products.expert_input_gradient(DY, W, _ends(3, 6))
    with pytest.raises(ValueError, match="requires cuda buffers"):
        products.expert_linear(X, W, _ends(3, 6))


def _saved(rows=6, columns=8, dtype=torch.float32):
    return products.ActivationCheckpoint(torch.zeros(rows, columns, dtype=torch.int8),
                                         torch.zeros(rows, -(-columns // 128), dtype=torch.uint8), dtype)


@pytest.mark.parametrize("arguments,message", [
    (dict(gradient=torch.zeros(5, 4)), "gradient has 5 rows, expected 6"),
    (dict(gradient=DY.half()), "x must use torch.float16"),
    (dict(x=_saved(dtype=torch.bfloat16)), "x must use torch.float32"),
    (dict(x=_saved(rows=5)), "gradient has 6 rows, expected 5"),
    (dict(x=_saved()._replace(exponents=torch.zeros(6, 2, dtype=torch.uint8))), "exponents has shape"),
    (dict(x=_saved()._replace(codes=torch.zeros(6, 8))), "codes and exponents must use int8 and uint8"),
    (dict(x=_saved()._replace(codes=torch.zeros(8, 6, dtype=torch.int8).T)), "codes must have contiguous rows"),
    (dict(x=_saved()._replace(dtype=torch.float64)), "dtype must be float32"),
    (dict(ends=_ends(3, 6).int()), "ends must use int64"),
    (dict(out_dtype=torch.bfloat16), "out_dtype must be torch.float32"),
    (dict(out=torch.zeros(4, 8)), "out must be 3D"),
    (dict(out=torch.zeros(4, 8).expand(2, 4, 8)), "matrices that do not overlap"),
    (dict(x=_saved()), "requires cuda buffers"),
    (dict(), "requires cuda buffers"),
])
def test_weight_gradient_refusals(arguments, message):
    call = dict(gradient=DY, x=X, ends=_ends(3, 6))
    call.update(arguments)
    with pytest.raises(ValueError, match=message):
        products.expert_weight_gradient(**call)


def test_checkpoint_and_int8_refusals():
    with pytest.raises(ValueError, match="requires cuda buffers"):
        products.checkpoint_activations(X)
    with pytest.raises(ValueError, match="x must use float32"):
        products.checkpoint_activations(X.int())
    with pytest.raises(ValueError, match="checkpoint must be an ActivationCheckpoint"):
        products.restore_activations(X)
    with pytest.raises(ValueError, match="out must use torch.float32"):
        products.restore_activations(_saved(), out=X.half())
    with pytest.raises(ValueError, match="requires cuda buffers"):
        products.restore_activations(_saved())
    with pytest.raises(ValueError, match="requires cuda buffers"):
        products.quantize_tokens(X)
    codes, scales = torch.zeros(6, 8, dtype=torch.int8), torch.zeros(6)
    weights, channels = torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4)
    for arguments, message in (
        ((codes.float(), scales, weights, channels), "codes must use int8"),
        ((codes, scales[:5], weights, channels), "6 rows and 5 scales"),
        ((codes, scales.double(), weights, channels), "scales must use float32"),
        ((codes, torch.zeros(12)[::2], weights, channels), "scales must be contiguous"),
        ((codes, scales, weights[:, :7], channels), "weight_codes have 7 columns, expected 8"),
        ((codes, scales, weights, channels), "requires cuda buffers"),
    ):
        with pytest.raises(ValueError, match=message):
            products.int8_product(*arguments)
    with pytest.raises(ValueError, match="out_dtype must be float32"):
        products.int8_product(codes, scales, weights, channels, out_dtype=torch.float64)
    long = torch.zeros(1, 131072, dtype=torch.int8)
    with pytest.raises(ValueError, match="131072 columns, at most 131071"):
        products.int8_product(long, torch.zeros(1), long, torch.zeros(1))


@pytest.mark.parametrize("name,arguments,message", [
    ("soapmi_expert_product", (3, P, 8, P, 8, 32, 0, P, 2, 6, 4, 8, 3, P, 4, 0, None), "dtype must be 0"),
    ("soapmi_expert_product", (1, P, 8, P, 8, 32, 0, P, 2, 6, 4, 8, 2, P, 4, 0, None), "out_dtype must be dtype or 0"),
    ("soapmi_expert_product", (0, P, 8, P, 8, 32, 0, P, 2, -1, 4, 8, 0, P, 4, 0, None), "non-negative"),
    ("soapmi_expert_product", (0, P, 8, P, 8, 32, 0, P, 2, 1 << 30, 4, 8, 0, P, 4, 0, None), "below 2\\^30"),
    ("soapmi_expert_product", (0, P, 8, P, 8, 32, 0, None, 2, 6, 4, 8, 0, P, 4, 0, None), "ends may be null"),
    ("soapmi_expert_product", (0, P, 7, P, 8, 32, 0, P, 2, 6, 4, 8, 0, P, 4, 0, None), "leading dimensions"),
    ("soapmi_expert_product", (0, P, 4, P, 8, 32, 1, P, 2, 6, 4, 8, 0, P, 4, 0, None), "leading dimensions"),
    ("soapmi_expert_product", (0, P, 8, P, 8, -1, 0, P, 2, 6, 4, 8, 0, P, 4, 0, None), "stride_w must be"),
    ("soapmi_expert_product", (0, P, 8, None, 8, 32, 0, P, 2, 6, 4, 8, 0, P, 4, 0, None), "nonzero"),
    ("soapmi_expert_weight_gradient", (0, P, 4, P, 8, P, 2, 6, 4, 8, 0, P, 8, 31, None, 0, None), "must not overlap"),
    ("soapmi_expert_weight_gradient", (0, P, 3, P, 8, P, 2, 6, 4, 8, 0, P, 8, 32, None, 0, None), "leading dimensions"),
    ("soapmi_expert_weight_gradient", (0, P, 4, None, 8, P, 2, 6, 4, 8, 0, P, 8, 32, None, 0, None), "nonzero"),
    ("soapmi_checkpoint_activations", (0, P, 8, 6, 8, P, 8, P, 0, None), "leading dimensions"),
    ("soapmi_checkpoint_activations", (0, None, 8, 6, 8, P, 8, P, 1, None), "nonzero"),
    ("soapmi_restore_activations", (7, P, 8, P, 1, 6, 8, P, 8, None), "dtype must be 0"),
    ("soapmi_quantize_rows", (0, P, 8, 6, 8, P, 7, P, None), "leading dimensions"),
    ("soapmi_quantize_rows", (0, P, 2000, 1 << 25, 2000, P, 2000, P, None), "too many rows"),
    ("soapmi_expert_product", (1, P, 8, P, 8, 64, 0, P, 1 << 20, 1 << 29, 1 << 20, 8, 1, P, 1 << 20, 0, None), "too many tiles"),
    ("soapmi_int8_product", (P, 131072, P, P, 131072, P, 6, 4, 131072, 1, P, 4, None), "at most 131071"),
    ("soapmi_int8_product", (P, 8, None, P, 8, P, 6, 4, 8, 1, P, 4, None), "nonzero"),
])
def test_entry_points_refuse(name, arguments, message):
    with pytest.raises(ValueError, match=message):
        _native.call(name, *arguments)


@pytest.mark.parametrize("name,arguments", [
    ("soapmi_expert_product", (1, None, 8, None, 8, 32, 0, P, 0, 0, 4, 8, 1, None, 4, 1, None)),
    ("soapmi_expert_product", (1, None, 8, None, 8, 0, 0, None, 1, 6, 0, 8, 1, None, 0, 1, None)),
    ("soapmi_expert_weight_gradient", (1, None, 4, None, 0, None, 1, 6, 4, 0, 1, None, 0, 0, None, 0, None)),
    ("soapmi_checkpoint_activations", (1, None, 8, 0, 8, None, 8, None, 1, None)),
    ("soapmi_restore_activations", (1, None, 0, None, 0, 0, 0, None, 0, None)),
    ("soapmi_quantize_rows", (1, None, 8, 0, 8, None, 8, None, None)),
    ("soapmi_int8_product", (None, 8, None, None, 8, None, 0, 4, 8, 1, None, 4, None)),
])
def test_empty_results_need_no_buffers(name, arguments):
    _native.call(name, *arguments)


LISTING = """
0000000000001000 <kernel>:
	s_load_dwordx2 s[0:1], s[4:5], 0x0                         // 000000001000: C0060002 00000000
	v_readfirstlane_b32 s{written}, v1                         // 000000001008: 7E080501
	{wait}                                                     // 00000000100C: BF800000
	s_cbranch_scc1 {jump}                                      // 000000001010: BF850001
	s_mov_b32 m0, s9                                           // 000000001014: BEFC0009
	s_nop 0                                                    // 000000001018: BF800000
	buffer_load_dwordx4 v2, s[0:3], s8 offen lds               // 00000000101C: E05D1000 08000002
	s_endpgm                                                   // 000000001024: BF810000
"""


@pytest.mark.parametrize("written,wait,jump,found", [
    (2, "s_nop 0", 4, 1), (8, "s_nop 0", 4, 1), (9, "s_nop 0", 4, 0), (2, "s_nop 1", 4, 0), (2, "s_nop 0", 65535, 1),
    (2, "s_nop 1", 2, 1),  # straight to the load
    (2, "s_nop 3", 2, 0),
])
def test_the_build_sees_a_load_that_does_not_wait(written, wait, jump, found):
    """The loads to LDS written in assembly are out of the compiler's sight: five wait states have to pass between
    a vector instruction that writes a scalar register and a memory instruction that reads it."""
    assert len(build.unsettled_loads(LISTING.format(written=written, wait=wait, jump=jump))) == found


@pytest.mark.parametrize("writer,found", [
    ("v_readlane_b32 s3, v1, 0", 1), ("v_cmp_gt_i32_e64 s[2:3], v1, s8", 1), ("v_cmp_gt_i32_e32 vcc, s2, v1", 0),
    ("v_mad_u64_u32 v[4:5], s[2:3], s0, v1, v[6:7]", 1), ("v_add_co_u32 v1, s[8:9], v2, v3", 1), ("v_add_u32_e32 v1, s8, v2", 0),
    ("s_add_i32 s8, s9, 4", 0)])
def test_the_build_sees_every_kind_of_writer(writer, found):
    line = LISTING.format(written=2, wait="s_nop 0", jump=4).replace("v_readfirstlane_b32 s2, v1", writer)
    assert len(build.unsettled_loads(line)) == found


def test_no_load_of_the_library_reads_a_register_too_soon():
    assert build.check_loads(_native.LIBRARY_PATH) > 100


@pytest.mark.skipif(torch.cuda.is_available(), reason="the launch has to fail for want of a GPU")
@pytest.mark.parametrize("name,arguments", [
    # rows, outputs, inputs: short inner sizes with many rows, on tiles straight from memory and through registers
    *(("soapmi_expert_product", (dtype, P, k, P, k, 0, 0, None, 1, tokens, n, k, dtype, P, n, 0, None))
      for dtype, tokens, n, k in ((1, 1 << 21, 4096, 8), (1, 1 << 21, 4096, 9), (1, 1 << 21, 4096, 10), (1, 1 << 21, 4096, 16),
                                  (1, 1 << 23, 1024, 8), (1, 1 << 28, 32, 16), (0, 1 << 21, 4096, 8), (0, 1 << 21, 4096, 16))),
    ("soapmi_int8_product", (P, 16, P, P, 16, P, 1 << 21, 4096, 16, 1, P, 4096, None)),
    # a million experts with a small matrix each
    ("soapmi_expert_weight_gradient", (1, P, 8, P, 8, P, 1 << 20, 1 << 26, 8, 8, 1, P, 8, 64, None, 0, None)),
])
def test_a_product_that_some_tile_can_take_is_launched(name, arguments):
    """The tile is chosen among those whose launch has fewer than 2^32 threads."""
    with pytest.raises(RuntimeError, match="kernel launch failed"):
        _native.call(name, *arguments)


def test_out_does_not_require_a_gradient():
    codes, scales = torch.zeros(6, 8, dtype=torch.int8), torch.zeros(6)

    def calls(out):
        return (lambda: products.expert_product(X, torch.zeros(8, 8), None, out=out),
                lambda: products.expert_input_gradient(X, torch.zeros(8, 8), None, out=out),
                lambda: products.expert_weight_gradient(torch.zeros(9, 6), torch.zeros(9, 8), None, out=out),
                lambda: products.restore_activations(_saved(), out=out),
                lambda: products.int8_product(codes, scales, torch.zeros(8, 8, dtype=torch.int8), torch.zeros(8), out=out))

    for call in calls(torch.zeros(6, 8, requires_grad=True)):
        with pytest.raises(ValueError, match="out must not require a gradient"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="requires cuda buffers"):
            call()


@pytest.mark.parametrize("experts,tokens,n,k", [
    (1, 1 << 20, 318550919442291584, 632734031689253760),  # as many tiles as 1 in 64 bits
    (1, 1 << 40, 64, 64), ((1 << 30) - 1, (1 << 30) - 1, (1 << 30) - 1, (1 << 30) - 1), (64, 1 << 20, 256, 256), (129, 1 << 20, 8, 8),
    (0, 1 << 20, 8, 8), (1, 1 << 20, -8, 8), (1, 1023, 8, 8)])
def test_no_workspace_where_sums_stay_whole(experts, tokens, n, k):
    assert _native.library().soapmi_expert_weight_gradient_workspace_bytes(experts, tokens, n, k) == 0


@pytest.mark.parametrize("experts,tokens,n,k,parts", [(1, 1 << 20, 8, 8, 256), (128, 1 << 20, 8, 8, 2), (2, 2048, 300, 500, 2),
                                                      (1, 6000, 72, 80, 11), (1, 1024, 8, 8, 2)])
def test_workspace_of_cut_sums(experts, tokens, n, k, parts):
    assert _native.library().soapmi_expert_weight_gradient_workspace_bytes(experts, tokens, n, k) == parts * experts * n * k * 4
