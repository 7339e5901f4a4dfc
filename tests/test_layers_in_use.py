"""The 8-bit layers' operators as programs use them beyond a plain call: saved-tensor
hooks, derivatives that are not there, captured graphs, streams, and a model's layers
made of them together.  Tests that need no GPU put a recorder in the place of the
library call."""

import pytest
import torch

from conftest import announce
from oracle import layers as ol

E8M0 = torch.float8_e8m0fnu


class _Library:
    """Stands for a case's library: an entry is its name."""

    def __getattr__(self, name):
        return name


@pytest.fixture
def recorded(monkeypatch):
    """[(entry, arguments)] of the calls that the operators would make, on CPU tensors."""
    import cases.block_matmul.op as matmul
    import cases.block_quant.op as quant
    import cases.rms_norm.op as norm
    from framework import capi
    calls = []

    def launch(entry, device, *args):
        calls.append((entry, args))
        return 0
    monkeypatch.setattr(capi, "launch", launch)
    require = capi.require
    monkeypatch.setattr(capi, "require", lambda cond, msg: require(cond or "GPU tensor" in msg, msg))
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    for op in (matmul, quant, norm):
        monkeypatch.setattr(op, "_lib", _Library)
    monkeypatch.setattr(norm, "_workspace_bytes", lambda *a: 1024)
    monkeypatch.setattr(matmul, "_workspace_bytes", lambda *a: 0)
    monkeypatch.setattr(matmul, "_layer_bytes", lambda *a: (1024, 1024, 512))
    return calls


def _norm(x, w):
    from cases.rms_norm.op import rms_norm
    return rms_norm(x, w)


def _summed(x, w):
    from cases.rms_norm.op import rms_norm
    y, h = rms_norm(x, w, x)
    return y + h


def _linear(x, w):
    from cases.block_matmul.op import block_linear
    return block_linear(x, w.expand(5, -1) if w.dim() == 1 else w)


def _prepared(x, w):
    from cases.block_matmul.op import block_linear, quantize_weight
    w = w.expand(5, -1) if w.dim() == 1 else w
    return block_linear(x, w, quantize_weight(w))


CALLS = {"rms_norm": _norm, "with_residual": _summed, "linear": _linear, "prepared": _prepared}


def _view(layout, base):
    return {"whole": base, "every_other": base[::2], "columns": base[:, ::2], "next": base[:-1],
            "expanded": base[:1].expand(7, -1), "transposed": base.t()}[layout]


LAYOUTS = ["whole", "every_other", "columns", "next", "expanded", "transposed"]


# ------------------------------------------------ tensors that hooks put elsewhere
@pytest.mark.parametrize("layout", LAYOUTS)
def test_backward_reads_the_saved_tensor_as_it_lies(layout, recorded):
    """Hooks may return a dense copy of what was saved as a view: the backward's strides are those
    of the copy, and its rows within it."""
    base = torch.randn(8, 12, requires_grad=True)
    x = _view(layout, base)
    w = torch.randn(x.size(1), requires_grad=True)
    packed = []

    def pack(t):
        packed.append(t.detach().clone(memory_format=torch.contiguous_format))
        return len(packed) - 1
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda i: packed[i]):
        y = _norm(x, w)
    y.backward(torch.ones_like(y))
    (entry, args), = [c for c in recorded if c[0].endswith("_backward")]
    copy, = [t for t in packed if t.data_ptr() == args[3]]
    assert copy.shape == x.shape and args[5] == copy.stride(0)
    rows, D = args[14:16]
    assert (rows, D) == x.shape and (rows - 1) * args[5] + D <= copy.numel()
    assert base.grad.shape == base.shape and w.grad.shape == w.shape


@pytest.mark.parametrize("name", CALLS)
def test_other_tensors_than_were_saved_are_refused(name, recorded):
    """A hook that returns another tensor, here one row or number short, is refused before a
    launch."""
    for which in range({"rms_norm": 3, "with_residual": 3, "linear": 1, "prepared": 3}[name]):
        x, w = torch.randn(6, 16, requires_grad=True), torch.randn(16, requires_grad=True)
        packed = []

        def pack(t):
            packed.append(t.detach())
            return len(packed) - 1

        def unpack(i):
            t = packed[i]
            return t[:-1] if i == which else t
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            out = CALLS[name](x, w)
        assert which < len(packed)
        del recorded[:]
        with pytest.raises(RuntimeError, match="saved"):
            out.backward(torch.ones_like(out))
        assert not [c for c in recorded if "backward" in c[0]]


@pytest.mark.parametrize("name,which", [("rms_norm", 2), ("with_residual", 0), ("with_residual", 2),
                                        ("linear", 0), ("prepared", 2)])
def test_other_types_than_were_saved_are_refused(name, which, recorded):
    """A hook that gives back fewer bytes: what would be read past them is refused."""
    x, w = torch.randn(6, 16, requires_grad=True), torch.randn(16, requires_grad=True)
    packed = []

    def pack(t):
        packed.append(t.detach())
        return len(packed) - 1

    def unpack(i):
        t = packed[i]
        return t if i != which else t.to(torch.bfloat16 if t.dtype == torch.float32 else torch.bool)
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        out = CALLS[name](x, w)
    assert which < len(packed)
    del recorded[:]
    with pytest.raises(RuntimeError, match="saved"):
        out.backward(torch.ones_like(out))
    assert not [c for c in recorded if "backward" in c[0]]


@pytest.mark.gpu
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("name", CALLS)
def test_gradients_of_offloaded_tensors(name, layout):
    announce(f"{name} offloaded {layout}")
    g = torch.Generator().manual_seed(1)
    base = torch.randn(40, 52, generator=g).cuda().requires_grad_(True)
    k = _view(layout, base).size(1)
    w = torch.randn(*((k,) if "linear" not in name and name != "prepared" else (9, k)),
                    generator=g).cuda().requires_grad_(True)
    out = CALLS[name](_view(layout, base), w)
    up = torch.randn(out.shape, generator=g).cuda()
    want = torch.autograd.grad(out, (base, w), up)
    with torch.autograd.graph.save_on_cpu():
        out = CALLS[name](_view(layout, base), w)
    got = torch.autograd.grad(out, (base, w), up)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


# ------------------------------------------------------------- version counters
def _overwritten_inputs_are_noticed(device):
    for name in ("rms_norm", "with_residual"):
        x = torch.randn(4, 16, device=device, requires_grad=True)
        w = torch.randn(16, device=device, requires_grad=True)
        h = x * 1.0
        out = CALLS[name](h, w)
        if name == "rms_norm":
            h.mul_(2.0)
        with torch.no_grad():
            w.add_(1.0)
        with pytest.raises(RuntimeError, match="inplace"):
            out.sum().backward()


def test_overwritten_inputs_are_noticed(recorded):
    _overwritten_inputs_are_noticed("cpu")


@pytest.mark.gpu
def test_inputs_overwritten_on_the_gpu_are_noticed():
    announce("rms_norm, version counters")
    _overwritten_inputs_are_noticed("cuda")


@pytest.mark.gpu
def test_a_weight_updated_between_forward_and_backward():
    """The layer keeps its own copy in 8 bits: the gradient is that of the forward."""
    from cases.block_matmul.op import block_linear
    announce("block_linear, weight updated before its backward")
    x = torch.randn(20, 300, device="cuda", requires_grad=True)
    w = torch.randn(40, 300, device="cuda", requires_grad=True)
    up = torch.randn(20, 40, device="cuda")
    want = torch.autograd.grad(block_linear(x, w), (x, w), up)
    y = block_linear(x, w)
    with torch.no_grad():
        w.add_(1.0)
        x.mul_(3.0)
    got = torch.autograd.grad(y, (x, w), up)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


# ---------------------------------------------------- derivatives that are not there
def _tangents_are_refused(name, device):
    import torch.autograd.forward_ad as forward_ad
    x = torch.randn(5, 16, device=device)
    w = torch.randn(*((16,) if "linear" not in name and name != "prepared" else (9, 16)),
                    device=device)
    with forward_ad.dual_level():
        for dual in (0, 1):
            args = [x, w]
            args[dual] = forward_ad.make_dual(args[dual], torch.ones_like(args[dual]))
            with pytest.raises(NotImplementedError):
                CALLS[name](*args)
            with torch.no_grad(), pytest.raises(NotImplementedError):
                CALLS[name](*args)
        CALLS[name](x, w)


@pytest.mark.parametrize("name", ["rms_norm", "with_residual", "linear"])
def test_tangents_are_refused(name, recorded):
    _tangents_are_refused(name, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["rms_norm", "with_residual", "linear"])
def test_tangents_on_the_gpu_are_refused(name):
    announce(f"{name} with a tangent")
    _tangents_are_refused(name, "cuda")


def _second_derivatives_are_refused(name, device):
    x = torch.randn(6, 16, device=device, requires_grad=True)
    w = torch.randn(*((16,) if "linear" not in name and name != "prepared" else (9, 16)),
                    device=device, requires_grad=True)
    for leaf in (x, w):
        out = CALLS[name](x, w).sum()
        (grad,) = torch.autograd.grad(out, leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="second"):
            (out + grad.square().sum()).backward()
    CALLS[name](x, w).sum().backward(create_graph=True)      # fine where nobody goes on from it
    (grad,) = torch.autograd.grad(CALLS[name](x, w).sum(), x)
    assert not grad.requires_grad


@pytest.mark.filterwarnings("ignore:Using backward")
@pytest.mark.parametrize("name", CALLS)
def test_second_derivatives_are_refused(name, recorded):
    _second_derivatives_are_refused(name, "cpu")


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore:Using backward")
@pytest.mark.parametrize("name", CALLS)
def test_second_derivatives_on_the_gpu_are_refused(name):
    announce(f"{name} differentiated twice")
    _second_derivatives_are_refused(name, "cuda")


def test_quantised_operators_refuse_gradients(recorded):
    from cases.block_matmul.op import block_matmul
    from cases.rms_norm.op import rms_norm_quantized
    x, w = torch.randn(3, 16, requires_grad=True), torch.randn(16)
    with pytest.raises(RuntimeError, match="no gradient"):
        rms_norm_quantized(x, w)
    with torch.no_grad():
        codes, scales = rms_norm_quantized(x, w)
    with pytest.raises(RuntimeError, match="no gradient"):
        block_matmul(codes, scales.float().requires_grad_(True), codes, scales.float())


# ------------------------------------------------------------------ captured graphs
def _replayed(make, run):
    """Captures run(inputs) and replays it on new inputs, with eager work between; every replay
    against the eager call.  A second graph of the same pool is replayed in turn."""
    static = [make(s) for s in (0, 1)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in static:
            run(s)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for s in static:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(run(s))
        graphs.append(g)
    for seed in range(2, 7):
        for i, (g, s, out) in enumerate(zip(graphs, static, outs)):
            new = make(seed + 10 * i)
            for a, b in zip(s, new):
                a.copy_(b)
            want = run(new)
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))
            (new[0].float() @ torch.ones(new[0].size(1), 3, device="cuda")).sum().item()


def _bits(tensors):
    return [t.view(torch.uint8) if "float8" in str(t.dtype) else t for t in tensors]


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["norm", "quant", "matmul", "long_matmul", "norm_train", "linear",
                                  "linear_train"])
def test_captured_and_replayed(what):
    from cases.block_matmul.op import block_linear, block_matmul
    from cases.block_quant.op import quantize_rows, quantize_tiles
    from cases.rms_norm.op import rms_norm, rms_norm_quantized
    announce(f"captured {what}")
    m, n, k = (100, 300, 6000) if what == "long_matmul" else (130, 200, 700)

    def make(seed):
        g = torch.Generator().manual_seed(seed)
        return [torch.randn(m, k, generator=g).cuda(), torch.randn(n, k, generator=g).cuda(),
                torch.randn(k, generator=g).cuda(), torch.randn(m, n, generator=g).cuda(),
                torch.randn(m, k, generator=g).cuda()]

    def run(t):
        x, w, v, up, dy = t
        if what == "norm":
            return _bits(rms_norm_quantized(x, v, dy)) + list(rms_norm(x, v, dy))
        if what == "quant":
            return _bits(quantize_rows(x, transposed=True)) + _bits(quantize_tiles(w, torch.float32,
                                                                                   transposed=True))
        if what.endswith("matmul"):
            a, b = quantize_rows(x), quantize_tiles(w)
            return [block_matmul(*a, *b), block_matmul(*a, *b, out_dtype=torch.float32)]
        if what == "linear":
            return [block_linear(x, w)]
        if what == "norm_train":
            x, v, dy = (a.detach().requires_grad_(True) for a in (x, v, dy))
            y, h = rms_norm(x, v, dy)
            return [y.detach(), h.detach()] + list(torch.autograd.grad((y, h), (x, v, dy),
                                                                       (t[0], t[4])))
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y = block_linear(x, w)
        return [y.detach()] + list(torch.autograd.grad(y, (x, w), up))
    _replayed(make, run)


# --------------------------------------------------------------- streams and devices
@pytest.mark.gpu
def test_calls_on_two_streams_at_once():
    """Each call's scratch is its own."""
    from cases.block_matmul.op import block_linear
    announce("block_linear on two streams")
    args = [[torch.randn(500, 4000, device="cuda"), torch.randn(300, 4000, device="cuda")]
            for _ in range(2)]
    want = [block_linear(*a) for a in args]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(block_linear(*args[i]))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


@pytest.mark.gpu
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_tensors_on_another_gpu_than_the_current_one():
    from cases.block_matmul.op import block_linear
    announce("block_linear on the second GPU")
    x, w = torch.randn(50, 300), torch.randn(40, 300)
    want = block_linear(x.cuda(0), w.cuda(0))
    got = block_linear(x.cuda(1), w.cuda(1))
    assert got.device.index == 1 and torch.equal(got.cpu(), want.cpu())
    with pytest.raises(RuntimeError):
        block_linear(x.cuda(0), w.cuda(1))


# ----------------------------------------------------------- the operators together
@pytest.mark.gpu
@pytest.mark.parametrize("scale_dtype", [torch.float32, E8M0], ids=str)
@pytest.mark.parametrize("d", [300, 2050, 5000, 17000])
def test_the_norm_quantises_as_the_quantiser_does(d, scale_dtype):
    """y in float32, quantised, is the norm's own output in 8 bits, to the last bit."""
    from cases.block_quant.op import quantize_rows
    from cases.rms_norm.op import rms_norm, rms_norm_quantized
    announce(f"rms_norm quantised apart {d} {scale_dtype}")
    g = torch.Generator().manual_seed(d)
    x, r, w = (torch.randn(*s, generator=g).cuda() for s in ((20, d), (20, d), (d,)))
    y, h = rms_norm(x, w, r)
    codes, scales, h2 = rms_norm_quantized(x, w, r, scale_dtype=scale_dtype)
    want = quantize_rows(y, scale_dtype)
    assert torch.equal(h, h2)
    assert all(torch.equal(a, b) for a, b in zip(_bits((codes, scales)), _bits(want)))


def _block(x, stream, params, scale_dtype):
    """A transformer's feed-forward layer: norm, two products, a gate, a product."""
    from cases.block_matmul.op import block_linear
    from cases.rms_norm.op import rms_norm
    norm, up, down = params
    y, stream = rms_norm(x, norm, stream)
    a, b = block_linear(y, up, scale_dtype=scale_dtype).chunk(2, -1)
    return block_linear(torch.nn.functional.silu(a) * b, down, scale_dtype=scale_dtype), stream


def _block64(x, stream, params, power2):
    norm, up, down = params
    y, stream, _ = ol.norm(x, norm, stream)
    q = lambda t, tiles=False: ol.values(*ol.quantize(t, tiles, power2))  # noqa: E731
    a, b = (q(y.float()) @ q(up, True).t()).chunk(2, -1)
    z = (torch.nn.functional.silu(a) * b).float()
    return q(z) @ q(down, True).t(), stream


@pytest.mark.gpu
@pytest.mark.parametrize("scale_dtype", [torch.float32, E8M0], ids=str)
@pytest.mark.parametrize("tokens", [1, 30])
def test_layers_of_a_model(tokens, scale_dtype):
    """Two layers and a head's token log-probabilities.  An intermediate result that falls on the
    other side of a rounding border moves by a step of four bits: the bound is on the whole, a
    step of 2^-3 for one number in a thousand, where the products' errors of 2^-20 reach one in
    about 10^5."""
    from cases.block_matmul.op import block_linear
    from cases.token_logp.op import token_logp
    announce(f"two layers, {tokens} tokens {scale_dtype}")
    g = torch.Generator().manual_seed(tokens)
    d, f, v = 320, 450, 1000

    def randn(*s, scale=1.0):
        return torch.randn(*s, generator=g) * scale
    params = [[1 + 0.1 * randn(d), randn(2 * f, d, scale=d ** -0.5), randn(d, f, scale=f ** -0.5)]
              for _ in range(2)]
    head, x, stream = randn(v, d, scale=d ** -0.5), randn(tokens, d), randn(tokens, d)
    labels = torch.randint(0, v, (tokens,), generator=g)
    a, b = x.cuda(), stream.cuda()
    wa, wb = x, stream
    with torch.no_grad():
        for p in params:
            a, b = _block(a, b, [t.cuda() for t in p], scale_dtype)
            wa, wb = _block64(wa, wb, p, scale_dtype != torch.float32)
            assert (a.cpu().double() - wa).norm() <= 2.0 ** -3 * 1e-3 ** 0.5 * wa.norm()
            wa, wb = a.cpu(), b.cpu()          # the next one from where this one stands
        logp = token_logp(block_linear(a + b, head.cuda(), scale_dtype=scale_dtype), labels.cuda())
    assert logp.shape == (tokens,) and torch.all(logp < 0)


@pytest.mark.gpu
def test_a_model_learns_to_its_gradients():
    """Forward and backward through two layers and a loss: every weight gets a finite gradient, and
    the whole step is bitwise repeatable."""
    from cases.block_matmul.op import block_linear
    from cases.token_logp.op import token_logp
    announce("training step of two layers")
    g = torch.Generator().manual_seed(5)
    d, f, v, tokens = 320, 450, 1000, 64

    def randn(*s, scale=1.0):
        return (torch.randn(*s, generator=g) * scale).bfloat16().cuda().requires_grad_(True)
    params = [[randn(d), randn(2 * f, d, scale=d ** -0.5), randn(d, f, scale=f ** -0.5)]
              for _ in range(2)]
    head, emb = randn(v, d, scale=d ** -0.5), randn(tokens, d)
    labels = torch.randint(0, v, (tokens,), generator=g).cuda()
    leaves = [t for p in params for t in p] + [head, emb]

    def step():
        x, stream = emb, torch.zeros(tokens, d, device="cuda")       # the stream in 32 bits
        for p in params:
            x, stream = _block(x, stream, p, E8M0)
        logits = block_linear((x + stream).bfloat16(), head)
        return torch.autograd.grad(-token_logp(logits, labels).mean(), leaves)
    first, second = step(), step()
    for t, a, b in zip(leaves, first, second):
        assert a.shape == t.shape and a.dtype == t.dtype
        assert torch.isfinite(a).all() and a.abs().max() > 0 and torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["rms_norm", "block_quant", "block_matmul"])
def test_the_case_passes_the_framework_s_own_check(name):
    import importlib

    from framework.verify import verify_all
    announce(f"verify_all {name}")
    case = importlib.import_module(f"cases.{name}").CASE
    op = importlib.import_module(f"cases.{name}.op")
    ok, report = verify_all(case, op.candidate, device="cuda")
    assert ok, report
