"""The training operators as programs use them beyond a plain call: the
precision that nobody asked for, autograd's hooks and version counters, saved
optimisers, operands that share memory.  Tests that need no GPU put a recorder
in the place of the library call."""

import pytest
import torch

from conftest import announce
from oracle import newton_schulz as ons


def _matrix(m, n, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = max(1, min(m, n) // 4)
    return (torch.randn(m, r, generator=g) @ torch.randn(r, n, generator=g) / r ** 0.5
            + 0.3 * torch.randn(m, n, generator=g))


# ------------------------------------------- Newton-Schulz: bits of the iterates
def _within_a_rounding(got, want, iterates, eps, factor=1.0):
    """got = want rounded to its type, `iterates` further off at most.  What roundings of the full
    iterates' size move the result by is in the norm: no element is off by more than all."""
    slack = factor * 4 * iterates.norm()
    assert torch.all((got.cpu().double() - want).abs() <= eps * 1.01 * want.abs() + slack + 2.0 ** -25)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,eps", [(torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)])
@pytest.mark.parametrize("m,n", [(150, 200), (300, 130)])
def test_16_bit_matrices_are_iterated_in_full(m, n, dtype, eps):
    from cases.newton_schulz.op import newton_schulz
    announce(f"newton_schulz of 16 bits, no precision given {m} x {n} {dtype}")
    G = _matrix(m, n).to(dtype)
    got = newton_schulz(G.cuda())
    assert torch.equal(got, newton_schulz(G.cuda(), precision="full"))
    want = ons.orthogonalise(G)
    off = ons.by_products(G, operand=2.0 ** -21, product=2.0 ** -22, seed=1)
    _within_a_rounding(got, want, off - want, eps)


@pytest.mark.gpu
def test_16_bit_weights_are_updated_from_full_iterates():
    from cases.newton_schulz.op import muon_step
    announce("muon_step of 16-bit weights, no precision given")
    W, G = (0.02 * _matrix(150, 200, 1)).bfloat16(), _matrix(150, 200, 2)
    Wd, Md = W.cuda(), torch.zeros(150, 200, device="cuda")
    full, Mf = W.cuda(), Md.clone()
    muon_step(Wd, G.cuda(), Md, lr=0.05, nesterov=False)
    muon_step(full, G.cuda(), Mf, lr=0.05, nesterov=False, precision="full")
    assert torch.equal(Wd, full)
    O = ons.orthogonalise(G)
    off = ons.by_products(G, operand=2.0 ** -21, product=2.0 ** -22, seed=1) - O
    _within_a_rounding(Wd, W.double() - 0.05 * O, off, 2.0 ** -8, 0.05)


# ---------------------------------------------------- a recorder for the library
class _Library:
    """Stands for a case's library: an entry is its name."""

    def __getattr__(self, name):
        return name


@pytest.fixture
def recorded(monkeypatch):
    """[(entry, arguments)] of the calls that the row operators would make, on CPU tensors."""
    import cases.policy_loss.op as policy
    import cases.preference_loss.op as preference
    import cases.token_logp.op as logp
    from framework import capi, token_rows
    calls = []

    def launch(entry, device, *args):
        calls.append((entry, args))
        return 0
    monkeypatch.setattr(capi, "launch", launch)
    monkeypatch.setattr(token_rows, "check", lambda *a: None)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    for op in (logp, policy, preference):
        monkeypatch.setattr(op, "_lib", _Library)
    for op in (policy, preference):
        monkeypatch.setattr(op, "_workspace_bytes", lambda *a: 1024)
    return calls


def _call(name, logits, labels):
    """The differentiable answer of an operator."""
    if name == "token_logp":
        from cases.token_logp.op import token_logp
        return token_logp(logits, labels).sum()
    zeros = torch.zeros(labels.shape, device=labels.device)
    if name == "policy_loss":
        from cases.policy_loss.op import policy_loss
        return policy_loss(logits, labels, zeros, zeros + 1.0)[0]
    from cases.preference_loss.op import preference_loss
    return preference_loss(logits, labels)[0]


NAMES = ["token_logp", "policy_loss", "preference_loss"]


def _view(layout, base):
    """A view of base [4, 6, V] whose rows are not one after the other."""
    return {"next_token": base[:, :-1], "every_other": base[:, ::2], "batch": base[::2],
            "expanded": base[:, :1].expand(-1, 5, -1), "sequence_first": base.transpose(0, 1)}[layout]


LAYOUTS = ["next_token", "every_other", "batch", "expanded", "sequence_first"]


# ------------------------------------------------ tensors that hooks put elsewhere
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("name", NAMES)
def test_backward_reads_the_saved_tensor_as_it_lies(name, layout, recorded):
    """Hooks may return a dense copy of what was saved as a view: the backward's strides are those
    of the copy, and its rows within it."""
    base = torch.randn(4, 6, 7, requires_grad=True)
    logits = _view(layout, base)
    labels = torch.zeros(logits.shape[:-1], dtype=torch.int64)
    packed = []

    def pack(t):
        packed.append(t.detach().clone(memory_format=torch.contiguous_format))
        return len(packed) - 1
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda i: packed[i]):
        out = _call(name, logits, labels)
    out.backward()
    (entry, args), = [c for c in recorded if c[0].endswith("_backward")]
    copy, = [t for t in packed if t.data_ptr() == args[0]]
    assert copy.shape == logits.shape
    at = 7     # before them: tensors, the type, the gradient that comes in
    assert args[at:at + 5] == (*logits.shape, copy.stride(0), copy.stride(1))
    B, S, V, bs, rs = args[at:at + 5]
    assert (B - 1) * bs + (S - 1) * rs + V <= copy.numel()
    assert base.grad.shape == base.shape


@pytest.mark.parametrize("name", NAMES)
def test_other_tensors_than_were_saved_are_refused(name, recorded):
    """A hook that returns another tensor, here one row short, is refused before a launch."""
    for which in range(3):              # logits, labels, statistics
        logits = torch.randn(4, 6, 7, requires_grad=True)
        labels = torch.zeros(4, 6, dtype=torch.int64)
        packed = []

        def pack(t):
            packed.append(t.detach())
            return len(packed) - 1

        def unpack(i):
            t = packed[i]
            return t[:-1] if i == which else t
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            out = _call(name, logits, labels)
        del recorded[:]
        with pytest.raises(RuntimeError, match="saved"):
            out.backward()
        assert not recorded


@pytest.mark.gpu
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("name", NAMES)
def test_gradients_of_offloaded_views(name, layout):
    announce(f"{name} offloaded {layout}")
    base = torch.randn(4, 6, 700, generator=torch.Generator().manual_seed(1)).cuda()
    base.requires_grad_(True)
    shape = _view(layout, base).shape[:-1]
    labels = torch.randint(0, 700, shape, generator=torch.Generator().manual_seed(2)).cuda()
    (want,) = torch.autograd.grad(_call(name, _view(layout, base), labels), base)
    with torch.autograd.graph.save_on_cpu():
        out = _call(name, _view(layout, base), labels)
    (got,) = torch.autograd.grad(out, base)
    assert torch.equal(got, want)


# ------------------------------------------------------------- version counters
def _in_place(logits):
    from cases.policy_loss.op import policy_loss_and_grad
    labels = torch.zeros(logits.shape[:-1], dtype=torch.int64, device=logits.device)
    zeros = torch.zeros(labels.shape, device=logits.device)
    loss, logp, dlogits = policy_loss_and_grad(logits, labels, zeros, zeros + 1.0, inplace=True)
    return dlogits


def _overwritten_logits_are_noticed(device):
    base = torch.randn(2, 3, 8, device=device, requires_grad=True)
    plain = base * 2.0
    at = plain._version
    plain.backward(_in_place(plain))         # the product did not keep its result
    assert plain._version > at and base.grad is not None
    for head in (torch.tanh, torch.exp, lambda t: torch.log_softmax(t, -1)):
        logits = head(base)
        with pytest.raises(RuntimeError, match="inplace"):
            logits.backward(_in_place(logits))
    logits = base * 2.0
    earlier = _call("token_logp", logits, torch.zeros(2, 3, dtype=torch.int64, device=device))
    _in_place(logits)
    with pytest.raises(RuntimeError, match="inplace"):
        earlier.backward()
    with torch.inference_mode():
        _in_place(torch.randn(2, 3, 8, device=device))


def test_overwritten_logits_are_noticed(recorded):
    _overwritten_logits_are_noticed("cpu")


@pytest.mark.gpu
def test_logits_overwritten_on_the_gpu_are_noticed():
    announce("policy_loss in place, version counters")
    _overwritten_logits_are_noticed("cuda")


@pytest.fixture
def recorded_updates(monkeypatch):
    """The same for muon_step, whose checks of devices are left out too."""
    import cases.newton_schulz.op as op
    from framework import capi
    calls = []

    def launch(entry, device, *args):
        calls.append((entry, args))
        return 0
    require = capi.require
    monkeypatch.setattr(capi, "launch", launch)
    monkeypatch.setattr(capi, "require", lambda cond, msg: require(cond or "one GPU" in msg, msg))
    monkeypatch.setattr(op, "_lib", _Library)
    monkeypatch.setattr(op, "_workspace_bytes", lambda *a: 1024)
    return calls


def _updated_weights_are_noticed(device):
    from cases.newton_schulz.op import Muon, muon_step
    x = torch.randn(5, 8, device=device)
    W = torch.nn.Parameter(torch.randn(8, 6, device=device))
    V = torch.nn.Parameter(torch.randn(6, 4, device=device))
    momenta = [torch.zeros(8, 6, device=device), torch.zeros(6, 4, device=device)]
    opt = Muon([W, V], lr=0.1)
    for step in (lambda: muon_step([W, V], [W.grad, V.grad], momenta, lr=0.1), opt.step):
        W.grad = V.grad = None
        out = (x @ W @ V).square().sum()
        out.backward(retain_graph=True)
        held = [W, V] + (momenta if step != opt.step else [opt.state[p]["momentum"]
                                                           for p in (W, V) if p in opt.state])
        before = [t._version for t in held]
        step()
        assert all(t._version > v for t, v in zip(held, before))
        with pytest.raises(RuntimeError, match="inplace"):
            out.backward()                      # the gradient of x @ W needs the old V


def test_updated_weights_are_noticed(recorded_updates):
    _updated_weights_are_noticed("cpu")


@pytest.mark.gpu
def test_weights_updated_on_the_gpu_are_noticed():
    announce("muon_step, version counters")
    _updated_weights_are_noticed("cuda")


# ---------------------------------------------------- derivatives that are not there
def _tangents_are_refused(name, device):
    import torch.autograd.forward_ad as forward_ad
    base = torch.randn(2, 3, 8, device=device)
    labels = torch.zeros(2, 3, dtype=torch.int64, device=device)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(base, torch.ones_like(base))
        with pytest.raises(NotImplementedError):
            _call(name, dual, labels)
        with torch.no_grad(), pytest.raises(NotImplementedError):
            _call(name, dual, labels)
        _call(name, base, labels)


@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_refused(name, recorded):
    _tangents_are_refused(name, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_tangents_on_the_gpu_are_refused(name):
    announce(f"{name} with a tangent")
    _tangents_are_refused(name, "cuda")


def _second_derivatives_are_refused(name, device):
    base = torch.randn(2, 3, 8, device=device, requires_grad=True)
    labels = torch.zeros(2, 3, dtype=torch.int64, device=device)
    for logits in (base, base[..., ::2]):        # read where they lie, and copied
        out = _call(name, logits, labels)
        (grad,) = torch.autograd.grad(out, base, create_graph=True)
        with pytest.raises(RuntimeError, match="second"):
            (out + grad.square().sum()).backward()
        out = _call(name, logits, labels)
        out.backward(create_graph=True)          # fine where nobody goes on from it
        base.grad = None
        out = _call(name, logits, labels)
        (grad,) = torch.autograd.grad(out, base)
        assert not grad.requires_grad


@pytest.mark.filterwarnings("ignore:Using backward")
@pytest.mark.parametrize("name", NAMES)
def test_second_derivatives_are_refused(name, recorded):
    _second_derivatives_are_refused(name, "cpu")


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore:Using backward")
@pytest.mark.parametrize("name", NAMES)
def test_second_derivatives_on_the_gpu_are_refused(name):
    announce(f"{name} differentiated twice")
    _second_derivatives_are_refused(name, "cuda")


# ------------------------------------------------------------- saved optimisers
def _momenta(opt):
    return [opt.state[p]["momentum"] for g in opt.param_groups for p in g["params"]
            if p in opt.state]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_a_loaded_optimiser_keeps_its_momenta(dtype):
    from cases.newton_schulz.op import Muon
    g = torch.Generator().manual_seed(5)

    def weights():
        return [torch.nn.Parameter(torch.zeros(4, 6, dtype=dtype)) for _ in range(3)]
    first = Muon([{"params": weights()}, {"params": weights(), "lr": 0.5}])
    for p in first.param_groups[0]["params"][:2] + first.param_groups[1]["params"]:
        first.state[p]["momentum"] = torch.randn(4, 6, generator=g)
    saved = first.state_dict()
    seen = []
    second = Muon([{"params": weights()}, {"params": weights()}])
    second.register_load_state_dict_post_hook(lambda o: seen.append([m.dtype for m in _momenta(o)]))
    second.load_state_dict(saved)
    assert seen == [[torch.float32] * 5] and second.param_groups[1]["lr"] == 0.5
    for a, b in zip(_momenta(first), _momenta(second)):
        assert torch.equal(a, b) and b.dtype == torch.float32
        assert a.data_ptr() != b.data_ptr()      # each updates its own
    # what hooks put in the place of the saved state counts; and a 16-bit momentum is widened
    third = Muon([{"params": weights()}, {"params": weights()}])

    def narrow(_, state):
        state["state"] = {k: {"momentum": v["momentum"].bfloat16()}
                          for k, v in state["state"].items()}
        return state
    third.register_load_state_dict_pre_hook(narrow)
    third.load_state_dict(first.state_dict())
    for a, b in zip(_momenta(first), _momenta(third)):
        assert b.dtype == torch.float32 and torch.equal(a.bfloat16().float(), b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_a_resumed_run_goes_on_as_it_was(dtype, tmp_path):
    from cases.newton_schulz.op import Muon
    announce(f"Muon saved and loaded {dtype}")
    g = torch.Generator().manual_seed(6)
    start = [(0.02 * torch.randn(s, generator=g)).to(dtype) for s in ((70, 90), (40, 30))]
    grads = [[torch.randn(p.shape, generator=g).to(dtype) for p in start] for _ in range(4)]

    def make(values):
        ps = [torch.nn.Parameter(v.cuda()) for v in values]
        return ps, Muon(ps, lr=0.05)

    def run(ps, opt, steps):
        for step in steps:
            for p, x in zip(ps, grads[step]):
                p.grad = x.cuda()
            opt.step()
    whole, opt = make(start)
    run(whole, opt, range(4))
    half, opt2 = make(start)
    run(half, opt2, range(2))
    torch.save({"weights": [p.detach() for p in half], "muon": opt2.state_dict()}, tmp_path / "at2")
    saved = torch.load(tmp_path / "at2", weights_only=True)
    resumed, opt3 = make(saved["weights"])
    opt3.load_state_dict(saved["muon"])
    run(resumed, opt3, range(2, 4))
    assert all(torch.equal(a, b) for a, b in zip(whole, resumed))
    assert all(torch.equal(a, b) for a, b in zip(_momenta(opt), _momenta(opt3)))


# ------------------------------------------------------ operands that share memory
def test_a_weight_listed_twice_is_refused_beside_empty_ones():
    from cases.newton_schulz.op import muon_step
    W, V, M, N, G = (torch.randn(4, 6) for _ in range(5))
    empty = torch.empty(0, 6)
    for weights, momenta in (([W, W], [M, N]), ([W, V], [M, M]), ([W, V], [V, N])):
        with pytest.raises(RuntimeError, match="twice"):
            muon_step(weights, [G, G], momenta, lr=0.1)
        with pytest.raises(RuntimeError, match="twice"):
            muon_step(weights + [empty], [G, G, empty], momenta + [empty], lr=0.1)


@pytest.mark.gpu
def test_empty_weights_are_passed_over():
    from cases.newton_schulz.op import muon_step
    announce("muon_step with empty weights")
    W, G, M = (torch.randn(4, 6, device="cuda") for _ in range(3))
    V, N = W.clone(), M.clone()
    empty = torch.empty(0, 6, device="cuda")
    muon_step([empty, W, empty], [empty, G, empty], [empty, M, empty], lr=0.1)
    muon_step(V, G, N, lr=0.1)
    assert torch.equal(W, V) and torch.equal(M, N)


def test_a_gradient_that_the_call_writes_is_refused(recorded_updates):
    """The momentum is stored before the gradient is read for the last time, and a weight while
    others' gradients still are."""
    from cases.newton_schulz.op import muon_step
    W, V, M, N, G, H = (torch.randn(6, 6) for _ in range(6))
    for grads in ([M, H], [G, M], [N, H], [V, H], [G, W]):
        with pytest.raises(RuntimeError, match="gradient shares"):
            muon_step([W, V], grads, [M, N], lr=0.1)
    assert not recorded_updates
    muon_step([W, V], [G, G], [M, N], lr=0.1)           # one gradient for both
    muon_step([W, V], [M.T, H], [M, N], lr=0.1)         # columns: copied before the first launch
    muon_step([W, V], [W, V], [M, N], lr=0.1)           # each read whole before it is written
    flat = torch.randn(6, 6 * 6)                        # columns of one buffer
    muon_step([flat[:, :6], flat[:, 6:12]], [flat[:, 12:18], flat[:, 18:24]],
              [flat[:, 24:30], flat[:, 30:]], lr=0.1)
    assert len(recorded_updates) == 4


# --------------------------------------------------------------- sizes and scalars
def test_more_pairs_than_a_launch_has_are_refused():
    import ctypes

    from test_capi import STATUS, _load
    lib = _load("cases.preference_loss.op")
    P = ctypes.c_void_p(1 << 20)                        # never dereferenced
    most = (2 ** 32 - 1) // 256                         # workgroups of 256, one a pair
    assert lib.preference_loss_workspace_bytes(1, 8, most) == 4 * (8 + most + 1)
    assert lib.preference_loss_workspace_bytes(1, 8, most + 1) == 0

    def call(pairs, cu, B, workspace_bytes):
        return lib.preference_loss_forward(P, 0, P, P, cu, pairs, P, P, P, P, B, 1, 8, 8, 8, -100,
                                           0.1, 0.0, 0, P, workspace_bytes, None)
    for cu, B in ((P, 1), (None, 2 * (most + 1))):
        assert call(most + 1, cu, B, 1 << 40) == STATUS["NL2K_ERR_OVERFLOW"]
        assert b"pairs" in lib.preference_loss_last_error()
    assert call(most, P, 1, 8) == STATUS["NL2K_ERR_WORKSPACE"]      # as many as that are taken


@pytest.mark.parametrize("denom", [1e-46, 1e39, 0.0, -1.0, float("nan"), float("inf")])
def test_a_denominator_that_32_bits_do_not_hold_is_refused(denom, recorded):
    from cases.policy_loss.op import policy_loss, policy_loss_and_grad
    logits, labels = torch.randn(2, 3, 8), torch.zeros(2, 3, dtype=torch.int64)
    zeros = torch.zeros(2, 3)
    for call in (policy_loss, policy_loss_and_grad):
        with pytest.raises(RuntimeError, match="denom"):
            call(logits, labels, zeros, zeros, denom=denom)
        call(logits, labels, zeros, zeros, denom=1e-40)
    assert len(recorded) == 2


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["one_token", "one_row", "one_sequence"])
def test_in_place_where_a_stride_stands_for_nothing(layout):
    """Contiguous logits whose dimensions of one element have strides of their own."""
    from cases.policy_loss.op import policy_loss_and_grad
    announce(f"policy_loss in place {layout}")
    base = torch.randn(1, 5, 40, generator=torch.Generator().manual_seed(3)).cuda()
    logits = {"one_token": base.transpose(0, 1),            # [5, 1, 40], strides 40, 200, 1
              "one_row": base[0, ::2][:1],                  # [1, 40], strides 80, 1
              "one_sequence": base.expand(3, 5, 40)[:1]}[layout]
    assert logits.is_contiguous()
    shape = logits.shape[:-1]
    labels = torch.randint(0, 40, shape, generator=torch.Generator().manual_seed(4)).cuda()
    old = torch.full(shape, -4.0, device="cuda")
    want = policy_loss_and_grad(logits, labels, old, old)
    got = policy_loss_and_grad(logits, labels, old, old, inplace=True)
    assert got[2].data_ptr() == logits.data_ptr()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.gpu
@pytest.mark.parametrize("v,dtype", [(2, torch.bfloat16), (3, torch.float32)])
def test_millions_of_rows_of_a_few_classes(v, dtype):
    """More rows than there are workgroups of 1024: a policy over a few actions."""
    from cases.policy_loss.op import policy_loss, policy_loss_and_grad
    rows = 2 ** 22 + 5
    announce(f"policy_loss {rows} rows of {v} {dtype}")
    g = torch.Generator(device="cuda").manual_seed(v)
    logits = torch.randn(rows, v, generator=g, device="cuda").to(dtype)
    labels = torch.randint(0, v, (rows,), generator=g, device="cuda")
    old = -torch.rand(rows, generator=g, device="cuda")
    adv = torch.randn(rows, generator=g, device="cuda")
    loss, logp, d = policy_loss_and_grad(logits, labels, old, adv, denom=1000.0)
    whole, lp = policy_loss(logits, labels, old, adv, denom=1000.0)
    assert torch.equal(loss, whole) and torch.equal(logp, lp)
    for part in (slice(0, 1000), slice(2 ** 21, 2 ** 21 + 1000), slice(rows - 1000, rows)):
        _, lp, dp = policy_loss_and_grad(logits[part], labels[part], old[part], adv[part],
                                         denom=1000.0)
        assert torch.equal(logp[part], lp) and torch.equal(d[part], dp)


# ------------------------------------------------------------ types and the case API
@pytest.mark.gpu
@pytest.mark.parametrize("how", ["step", "inplace", "train"])
@pytest.mark.parametrize("v", [1, 7, 33, 2050, 8190, 65540, 131080])
def test_policy_loss_of_float16(v, how):
    import test_gpu_policy_loss as policy
    announce(f"policy_loss float16, width {v} {how}")
    b, s = (3, 5) if v < 5000 else (2, 2)
    g, x, labels, old, ref, adv = policy._inputs(b, s, v, torch.float16)
    mask = torch.rand(b, s, generator=g) < 0.7
    mask[0, 0] = True
    labels[-1, -1] = policy.orow.IGNORE
    got = policy._run(x, labels, old, ref, adv, mask, 0.05, how)
    assert got[2].dtype == torch.float16
    policy._compare(x, labels, old, ref, adv, mask, 0.05, got)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES + ["newton_schulz"])
def test_the_case_passes_the_framework_s_own_check(name):
    import importlib

    from framework.verify import verify_all
    announce(f"verify_all {name}")
    case = importlib.import_module(f"cases.{name}").CASE
    op = importlib.import_module(f"cases.{name}.op")
    ok, report = verify_all(case, op.candidate, device="cuda")
    assert ok, report
