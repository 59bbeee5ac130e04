"""Activations in 8 bits against their definition, and what the expert linears' backward pass makes of them.

Every step of the definition is one FP32 operation, whose correctly rounded result a float64 operation rounded to FP32
gives as well, so codes, scales and values are compared bit for bit.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _definition(x):
    """(codes, scales, values) of finite x [rows, width], on the CPU."""
    rows, width = x.shape
    f = torch.nn.functional.pad(x.cpu().double(), (0, -width % 128)).view(rows, -1, 128)
    third = torch.tensor(1.0 / 127.0, dtype=torch.float64).float().double()
    scale = (f.abs().amax(2).clamp(min=2.0 ** -100) * third).float()
    inverse = (1.0 / scale.double()).float().double()
    codes = torch.round((f * inverse[..., None]).float()).clamp(-127, 127)
    values = (codes.double() * scale.double()[..., None]).float().to(x.dtype)
    return codes.view(rows, -1)[:, :width].to(torch.int8), scale, values.view(rows, -1)[:, :width]


def _rows(rows, width, dtype, device, seed=0):
    g = torch.Generator().manual_seed(seed + rows + 3 * width)
    x = torch.randn(rows, width, generator=g) * torch.exp2(8 * torch.randn(rows, 1, generator=g)).clamp(2 ** -12, 2 ** 12)
    return x.to(dtype).to(device)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [1, 2, 3, 4, 7, 8, 15, 16, 33, 64, 65, 127, 128, 129, 136, 250, 256, 512, 1021, 8192])
def test_codes_and_values(device, width, dtype):
    from ictc_o3 import decode_activations, encode_activations
    for rows in (1, 5, 127, 1025):
        x = _rows(rows, width, dtype, device)
        codes, scales = encode_activations(x)
        ref, ref_scales, ref_values = _definition(x)
        assert codes.dtype == torch.int8 and scales.dtype == torch.float32
        assert torch.equal(codes.cpu(), ref) and torch.equal(scales.cpu(), ref_scales)
        values = decode_activations(codes, scales, dtype=dtype)
        assert values.dtype == dtype and torch.equal(values.cpu(), ref_values)
        # half a scale, and FP32's roundings of the product, the scale and the value; then the type's
        full = decode_activations(codes, scales)
        step = scales.repeat_interleave(128, 1)[:, :width].double()
        assert ((full.double() - x.double()).abs() <= step * (0.5 + 127 * 2.0 ** -21)).all()


def test_any_shape_and_stride(device):
    from ictc_o3 import decode_activations, encode_activations
    x = _rows(24, 200, torch.bfloat16, device)
    codes, scales = encode_activations(x)
    for shape in ((2, 3, 4, 200), (24, 1, 200)):
        c, s = encode_activations(x.view(shape))
        assert c.shape == shape and s.shape == shape[:-1] + (2,)
        assert torch.equal(c.view(24, 200), codes) and torch.equal(s.view(24, 2), scales)
        assert torch.equal(decode_activations(c, s).view(24, 200), decode_activations(codes, scales))
    c, s = encode_activations(x[3])
    assert torch.equal(c, codes[3]) and torch.equal(s, scales[3])
    wide = torch.zeros(24, 311, dtype=torch.bfloat16, device=device)
    wide[:, 5:205] = x
    for same in (wide[:, 5:205], x.t().contiguous().t()):
        assert torch.equal(encode_activations(same)[0], codes)
    assert torch.equal(encode_activations(x[:1].expand(24, 200))[0], codes[:1].expand(24, 200))
    assert torch.equal(decode_activations(codes.t().contiguous().t(), scales.t().contiguous().t()),
                       decode_activations(codes, scales))
    none = torch.empty(0, 70, device=device)
    c, s = encode_activations(none)
    assert c.shape == (0, 70) and s.shape == (0, 1) and decode_activations(c, s).shape == (0, 70)


def test_zeros_small_large_and_bad_values(device):
    from ictc_o3 import decode_activations, encode_activations
    x = torch.zeros(8, 300, device=device)
    g = torch.Generator().manual_seed(1)
    noise = torch.randn(300, generator=g).to(device)
    x[1], x[2] = noise * 2.0 ** -110, noise * 2.0 ** -140          # below the least scale
    x[3] = (noise / noise.abs().max()).clamp(-1, 1) * 3.4e38
    x[4], x[5] = noise, noise
    x[4, 140], x[5, 299] = float("nan"), float("-inf")
    x[6] = -noise * 2.0 ** -99
    ok = [0, 1, 2, 3, 6, 7]
    codes, scales = encode_activations(x)
    ref, ref_scales, ref_values = _definition(x[ok])
    assert torch.equal(codes[ok].cpu(), ref) and torch.equal(scales[ok].cpu(), ref_scales)
    values = decode_activations(codes, scales)
    assert torch.equal(values[ok].cpu(), ref_values) and (values[0] == 0).all() and (values[2] == 0).all()
    bad = torch.zeros(2, 300, dtype=torch.bool, device=device)
    bad[0, 128:256], bad[1, 256:] = True, True
    assert torch.equal(values[4:6].isnan(), bad)
    assert torch.equal(values[4, :128], decode_activations(*encode_activations(noise))[:128])


def test_offsets_past_32_bits(device):
    from ictc_o3 import decode_activations, encode_activations
    x = torch.zeros(34000001, 64, dtype=torch.bfloat16, device=device)
    x[-300:] = _rows(300, 64, torch.bfloat16, device)
    codes, scales = encode_activations(x)
    ref, ref_scales, ref_values = _definition(x[-300:])
    assert torch.equal(codes[-300:].cpu(), ref) and torch.equal(scales[-300:].cpu(), ref_scales)
    assert (codes[:-300] == 0).all()
    del x
    values = decode_activations(codes, scales, dtype=torch.bfloat16)
    assert torch.equal(values[-300:].cpu(), ref_values) and (values[:-300] == 0).all()


def test_refusals(device):
    from ictc_o3 import decode_activations, encode_activations, expert_linear, expert_order
    x = torch.zeros(4, 200, device=device)
    codes, scales = encode_activations(x)
    for call, match in ((lambda: encode_activations(x.double()), "float32"),
                        (lambda: encode_activations(x[:, :0]), "last axis"),
                        (lambda: encode_activations(x[0, 0]), "last axis"),
                        (lambda: decode_activations(codes, scales[:, :1]), "scales"),
                        (lambda: decode_activations(codes, scales.double()), "scales"),
                        (lambda: decode_activations(codes, scales.cpu()), "scales"),
                        (lambda: decode_activations(codes.view(torch.uint8), scales), "int8"),
                        (lambda: decode_activations(codes, scales, dtype=torch.float64), "dtype"),
                        (lambda: expert_linear(x, torch.zeros(1, 3, 200, device=device),
                                               expert_order(torch.zeros(4, dtype=torch.int64, device=device), 1),
                                               save_bits=4), "save_bits")):
        with pytest.raises(ValueError, match=match):
            call()


def _linear(rows, experts, inputs, outputs, dtype, device):
    g = torch.Generator().manual_seed(rows + inputs)
    x = torch.randn(rows, inputs, generator=g).to(dtype).to(device)
    W = (torch.randn(experts, outputs, inputs, generator=g) / inputs ** 0.5).to(dtype).to(device)
    b, gy = (torch.randn(n, outputs, generator=g).to(dtype).to(device) for n in (experts, rows))
    ids = torch.randint(-1, experts, (rows,), generator=g).to(device)
    return x, W, b, gy, ids


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,experts,inputs,outputs", [(0, 2, 8, 8), (1, 3, 16, 5), (70, 4, 7, 33), (300, 10, 128, 128),
                                                         (5000, 3, 200, 333), (4096, 2, 512, 256), (999, 1, 1, 1),
                                                         (2000, 7, 136, 72), (20000, 10, 264, 128), (60000, 3, 520, 264),
                                                         (333, 90, 128, 64), (7, 1, 8, 8)])
def test_expert_linear(device, rows, experts, inputs, outputs, dtype):
    """Result and row gradient are those of whole rows, bit for bit; the weights' and biases' gradients those that the
    decoded rows have."""
    from ictc_o3 import decode_activations, encode_activations, expert_linear, expert_order
    x, W, b, gy, ids = _linear(rows, experts, inputs, outputs, dtype, device)
    order = expert_order(ids, experts)
    value = decode_activations(*encode_activations(x), dtype=dtype)
    for t in (x, value, W, b):
        t.requires_grad_()
    y, whole = expert_linear(x, W, order, b, save_bits=8), expert_linear(x, W, order, b)
    got, ref = (torch.autograd.grad(t, (x, W, b), gy) for t in (y, whole))
    from_value = torch.autograd.grad(expert_linear(value, W, order, b), (W, b), gy)
    assert torch.equal(y, whole) and torch.equal(got[0], ref[0])
    assert torch.equal(got[1], from_value[0]) and torch.equal(got[2], from_value[1])


def test_expert_linear_gradients_of_gradients(device):
    """The derivative of the weights' gradient passes through the codes to the rows, as that of whole rows does."""
    from ictc_o3 import decode_activations, encode_activations, expert_linear, expert_order
    x, W, b, gy, ids = _linear(400, 5, 96, 80, torch.float32, device)
    order = expert_order(ids, 5)
    value = decode_activations(*encode_activations(x))
    for t in (x, value, W, b, gy):
        t.requires_grad_()
    cots = [torch.randn_like(t) for t in (x, W, b)]
    out = []
    for rows, bits in ((x, 8), (value, None)):
        first = torch.autograd.grad(expert_linear(rows * 1.0, W, order, b, save_bits=bits), (rows, W, b), gy, create_graph=True)
        out.append((*first, *torch.autograd.grad(first, (rows, W, gy), cots)))
    assert all(torch.equal(i, j) for i, j in zip(*out))


def test_expert_linear_keeps_a_byte_an_element(device):
    from ictc_o3 import expert_linear, expert_order
    rows, width = 65536, 256
    ids = torch.zeros(rows, dtype=torch.int64, device=device)
    order = expert_order(ids, 1)
    base = torch.randn(rows, width, device=device, requires_grad=True)
    W = torch.randn(1, 8, width, device=device)

    def kept(bits, weight):
        before = torch.cuda.memory_allocated()
        y = expert_linear(base * 2.0, weight, order, save_bits=bits)
        return torch.cuda.memory_allocated() - before - y.numel() * 4

    full, eight = (kept(bits, W.clone().requires_grad_()) for bits in (None, 8))
    slack = 1 << 20
    assert full > rows * width * 4 - slack and eight < rows * (width + 8) + slack
    assert kept(8, W) > full - slack      # (the rows are not needed, and whole ones are kept as without the argument)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_a_function_that_keeps_its_input_in_8_bits(device, dtype):
    """A caller's own backward pass: the gradient is its formula at the decoded values, bit by bit."""
    from ictc_o3 import decode_activations, encode_activations

    class Gate(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            ctx.save_for_backward(*encode_activations(x))
            ctx.dtype = x.dtype
            return x * torch.tanh(x)

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, g):
            x = decode_activations(*ctx.saved_tensors, dtype=ctx.dtype)
            t = torch.tanh(x)
            return g * (t + x * (1 - t * t))

    generator = torch.Generator().manual_seed(8)
    x, g = (torch.randn(37, 5, 130, generator=generator).to(dtype).to(device) for _ in range(2))
    x.requires_grad_()
    y = Gate.apply(x)
    (got,) = torch.autograd.grad(y, x, g)
    d = decode_activations(*encode_activations(x), dtype=dtype)
    t = torch.tanh(d)
    assert torch.equal(got, g * (t + d * (1 - t * t))) and not torch.equal(d, x)


def test_longest_last_axis(device):
    """A row of 2^31 - 1 elements, the longest that is taken: its first, middle and last blocks against the definition."""
    from ictc_o3 import decode_activations, encode_activations
    width = 2 ** 31 - 1
    x = torch.zeros(1, width, dtype=torch.bfloat16, device=device)
    spans = [(0, 4096), (2 ** 30 - 1280, 2 ** 30 + 1280), (width - 4223, width)]   # (from whole blocks on)
    for k, (a, b) in enumerate(spans):
        x[:, a:b] = _rows(1, b - a, torch.bfloat16, device, k)
    codes, scales = encode_activations(x)
    assert codes.shape == (1, width) and scales.shape == (1, 2 ** 24)
    values = decode_activations(codes, scales, dtype=torch.bfloat16)
    for a, b in spans:
        ref, ref_scales, ref_values = _definition(x[:, a:b])
        assert torch.equal(codes[:, a:b].cpu(), ref) and torch.equal(values[:, a:b].cpu(), ref_values)
        assert torch.equal(scales[:, a // 128:(b + 127) // 128].cpu(), ref_scales)
    assert not codes[:, 4096:2 ** 30 - 1280].any() and not codes[:, 2 ** 30 + 1280:width - 4223].any()
