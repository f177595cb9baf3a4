"""flash_moba_rotary_func against the formula in 64 bits: values, gradients (the formula's, differences, the second
derivative), strides, streams and graphs.

Error of an output: it is rounded once (half a step, eps / 2 of its value; 2^-25 where fp16 is subnormal), from 32-bit products of cosine and
sine.  These are off by at most 2.2e-7: 2 pi 2^-26 for the fraction of a turn in 32 bits, 2^-23 for two units in the last place of the functions.  A
product and the sum add 2^-24 of (|x| + |y|) each: 5e-7 (|x| + |y|) covers all of it."""
import math

import pytest
import torch

import flash_moba

gpu = pytest.mark.gpu


def formula(x, positions, sections, base, rotary_dim, interleaved, sign=1.0):
    x = x.double()
    out, size = x.clone(), x.abs()
    j = 0
    for axis, count in enumerate(sections):
        for _ in range(count):
            angle = sign * positions[axis].double() * base ** (-2.0 * j / rotary_dim)
            c, s = angle.cos()[:, None], angle.sin()[:, None]
            a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + rotary_dim // 2)
            out[..., a] = x[..., a] * c - x[..., b] * s
            out[..., b] = x[..., a] * s + x[..., b] * c
            size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
            j += 1
    return out, size


def check(name, got, x, *args, sign=1.0, angle_error=0.0, dtype=None):
    want, size = formula(x, *args, sign=sign)
    err = (got.double() - want).abs()
    tol = want.abs() * torch.finfo(got.dtype).eps / 2 + size * (5e-7 + angle_error) + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    tol[..., args[3]:] = 0.0  # copied
    assert got.dtype == x.dtype and bool((err <= tol).all()), f"{name}: {(err - tol).max().item():.3e} over"


def make(tokens, heads, heads_k, dim, axes, far, dtype, seed, int64=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k, dq, dk = (torch.randn((tokens, h, dim), generator=g, device="cuda").to(dtype) for h in (heads, heads_k, heads, heads_k))
    positions = torch.randint(0, far, (axes, tokens), generator=g, device="cuda", dtype=torch.int64 if int64 else torch.int32)
    return q, k, dq, dk, positions


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,heads,heads_k,dim,rotary_dim,sections,interleaved", [
    (1, 1, 1, 8, 8, (4,), False),
    (1, 32, 8, 128, 128, (64,), False),
    (777, 8, 2, 128, 128, (16, 24, 24), False),
    (300, 4, 4, 128, 64, (8, 12, 12), True),
    (65, 3, 1, 80, 40, (20,), False),       # halves of 20: vectors of four
    (65, 3, 1, 80, 40, (7, 13), True),
    (130, 5, 5, 96, 96, (0, 1, 47), False),  # an axis without pairs
    (1030, 2, 2, 256, 256, (32, 32, 32, 32), False),
    (1030, 2, 1, 256, 8, (4,), True),
    (3001, 16, 16, 64, 64, (32,), False),
])
def test_values_and_gradients_are_the_formulas(dtype, tokens, heads, heads_k, dim, rotary_dim, sections, interleaved):
    q, k, dq, dk, pos = make(tokens, heads, heads_k, dim, len(sections), 1 << 18, dtype, 3, int64=dim == 96)
    form = (pos, sections, 10000.0, rotary_dim, interleaved)
    qg, kg = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
    qo, ko = flash_moba.flash_moba_rotary_func(qg, kg, pos, sections, rotary_dim=rotary_dim, interleaved=interleaved)
    check("q", qo.detach(), q, *form)
    check("k", ko.detach(), k, *form)
    gq, gk = torch.autograd.grad((qo, ko), (qg, kg), (dq, dk))
    check("dq", gq, dq, *form, sign=-1.0)
    check("dk", gk, dk, *form, sign=-1.0)
    with torch.no_grad():  # the same without a graph, and once more: no bit differs
        q1, k1 = flash_moba.flash_moba_rotary_func(q, k, pos, sections, rotary_dim=rotary_dim, interleaved=interleaved)
    assert torch.equal(q1, qo) and torch.equal(k1, ko) and not q1.requires_grad


@gpu
@pytest.mark.parametrize("base", [1.0, 500000.0])
def test_far_positions_and_bases(base):
    q, k, _, _, pos = make(64, 2, 2, 64, 1, 1 << 20, torch.float16, 5, int64=True)
    pos[0, :5] = torch.tensor([0, 1, (1 << 31) - 1, 1 << 31, -7])
    qo, ko = flash_moba.flash_moba_rotary_func(q, k, pos[0], base=base)
    # 2^31 / (2 pi) turns, each formed to 2^-50 of itself here and in the reference
    check("q", qo, q, pos, (32,), base, 64, False, angle_error=2 * math.pi * (2.0 ** 31 / 6.28) * 2.0 ** -49)


@gpu
def test_strided_inputs_are_read_where_they_lie():
    g = torch.Generator(device="cuda").manual_seed(8)
    qkv = torch.randn((333, 3, 4, 64), generator=g, device="cuda").to(torch.bfloat16)
    pos = torch.randint(0, 4000, (333, 2), generator=g, device="cuda").t()  # (strided positions too)
    q, k, _ = qkv.unbind(1)
    qo, ko = flash_moba.flash_moba_rotary_func(q, k, pos, (20, 12))
    assert qo.is_contiguous() and ko.is_contiguous()
    check("q", qo, q, pos, (20, 12), 10000.0, 64, False)
    check("k", ko, k, pos, (20, 12), 10000.0, 64, False)
    turned = qkv.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2)  # features not dense
    qt, kt = flash_moba.flash_moba_rotary_func(turned[:, 0], turned[:, 1], pos, (20, 12))
    assert torch.equal(qt, qo) and torch.equal(kt, ko)
    odd = torch.empty(333 * 4 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(333, 4, 64).copy_(q)  # not on 16 bytes
    assert torch.equal(flash_moba.flash_moba_rotary_func(odd, k, pos, (20, 12))[0], qo)
    one = q[:1, :1].expand(333, 4, 64)  # broadcast
    check("one", flash_moba.flash_moba_rotary_func(one, k, pos, (20, 12))[0], one, pos, (20, 12), 10000.0, 64, False)
    assert flash_moba.flash_moba_rotary_func(q[:0], k[:0], pos[:, :0], (20, 12))[0].shape == (0, 4, 64)


@gpu
def test_gradients_are_differences():
    """The turn is linear: <turn(q + h d) - turn(q), g> = h <d, grad>.  With h = 2^3 the roundings to 16 bits (2^-9 of an output of about 8, random in sign over
    64 * 2 * 64 terms) stay below a hundredth of h |d| |g| sqrt(terms)."""
    q, k, dq, dk, pos = make(64, 2, 2, 64, 1, 5000, torch.bfloat16, 9)
    qg = q.clone().requires_grad_(True)
    out = flash_moba.flash_moba_rotary_func(qg, k, pos)[0]
    grad, = torch.autograd.grad(out, qg, dq)
    d = torch.randn_like(q.float()).to(torch.bfloat16)
    more = (q.float() + 8 * d.float()).to(torch.bfloat16)
    with torch.no_grad():
        moved = flash_moba.flash_moba_rotary_func(more, k, pos)[0].double() - out.detach().double()
    got, want = (moved * dq.double()).sum().item(), ((more.double() - q.double()) * grad.double()).sum().item()
    assert abs(got - want) < 0.01 * 8 * math.sqrt(q.numel())


@gpu
def test_one_gradient_alone_second_derivatives_and_broadcast_gradients():
    q, k, dq, dk, pos = make(40, 2, 1, 64, 1, 5000, torch.float16, 10)
    qg = q.clone().requires_grad_(True)
    qo, ko = flash_moba.flash_moba_rotary_func(qg, k, pos)
    assert not k.requires_grad
    gq, = torch.autograd.grad(qo.sum(), qg)  # a gradient with strides of zero
    check("sum", gq, torch.ones_like(q), pos, (32,), 10000.0, 64, False, sign=-1.0)
    qo, _ = flash_moba.flash_moba_rotary_func(qg, k, pos)
    dqg = dq.clone().requires_grad_(True)
    gq, = torch.autograd.grad(qo, qg, dqg, create_graph=True)
    back, = torch.autograd.grad(gq, dqg, q)
    check("second", back, q, pos, (32,), 10000.0, 64, False)


@gpu
def test_other_streams_and_graphs():
    q, k, dq, dk, pos = make(500, 4, 2, 128, 3, 9000, torch.bfloat16, 11)
    sections = (16, 24, 24)

    def step(q, k):
        qo, ko = flash_moba.flash_moba_rotary_func(q, k, pos, sections)
        return (qo.detach(), ko.detach()) + torch.autograd.grad((qo, ko), (q, k), (dq, dk))  # (no graph of the leaves stays alive)

    qg, kg = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
    want = step(qg, kg)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(qg, kg)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(qg, kg)
    for i in range(3):
        with torch.no_grad():
            qg.copy_(q + i)
        graph.replay()
        torch.cuda.synchronize()
        want = step(qg, kg)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held)), i


@gpu
def test_a_leaf_of_a_living_eager_graph_is_not_captured():
    """The gradient's node of such a leaf belongs to the stream of the eager graph; a captured backward would draw that stream into the capture."""
    q, k, dq, dk, pos = make(50, 2, 2, 64, 1, 900, torch.bfloat16, 13)
    qg = q.clone().requires_grad_(True)
    alive = flash_moba.flash_moba_rotary_func(qg, k, pos)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="another stream and is still alive"):
        with torch.cuda.graph(graph):
            flash_moba.flash_moba_rotary_func(qg, k, pos)
    with torch.no_grad():
        want = flash_moba.flash_moba_rotary_func(qg, k, pos)
    assert torch.equal(alive[0].detach(), want[0])


@gpu
def test_compiled_and_in_front_of_the_training_function():
    """Positions, then gated attention, forward and backward, as a model calls them; the turn traced into a graph is the eager one."""
    q, k, dq, dk, pos = make(700, 4, 4, 64, 1, 700, torch.bfloat16, 12)
    pos[0] = torch.arange(700)
    v = torch.randn_like(k)
    cu = torch.tensor([0, 700], dtype=torch.int32, device="cuda")

    def model(q, k):
        q, k = flash_moba.flash_moba_rotary_func(q, k, pos)
        return flash_moba.flash_moba_varlen_func(q, k, v, cu, cu, 700, 700, 64, 3)

    qg, kg = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
    out = model(qg, kg)
    grads = torch.autograd.grad(out, (qg, kg), dq)
    q1, k1 = (x.detach().requires_grad_(True) for x in flash_moba.flash_moba_rotary_func(q, k, pos))
    out1 = flash_moba.flash_moba_varlen_func(q1, k1, v, cu, cu, 700, 700, 64, 3)
    g1 = torch.autograd.grad(out1, (q1, k1), dq)
    assert torch.equal(out, out1)
    for name, got, g in zip("qk", grads, g1):
        check(name, got, g, pos, (32,), 10000.0, 64, False, sign=-1.0)
    traced = torch.compile(lambda q, k: flash_moba.flash_moba_rotary_func(q, k, pos), backend="aot_eager", fullgraph=True)
    qo, ko = traced(qg, kg)
    e = flash_moba.flash_moba_rotary_func(qg, kg, pos)
    assert torch.equal(qo, e[0]) and torch.equal(ko, e[1])
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad((qo, ko), (qg, kg), (dq, dk)), torch.autograd.grad(e, (qg, kg), (dq, dk))))


@gpu
@pytest.mark.parametrize("change,message", [
    (dict(dtype=torch.float32), "fp16 and bf16"), (dict(rotary_dim=12), "rotary_dim"), (dict(rotary_dim=72), "rotary_dim"), (dict(sections=(31,)), "sections"),
    (dict(sections=(16, 16)), "axes"), (dict(base=0.5), "base"), (dict(base=math.inf), "base"), (dict(positions=torch.float32), "int32 or int64"),
    (dict(rows=3), "positions must have shape"), (dict(kdim=32), "same tokens"),
])
def test_refusals(change, message):
    q = torch.zeros((4, 2, 64), dtype=change.get("dtype", torch.bfloat16), device="cuda")
    k = q[..., :change.get("kdim", 64)]
    pos = torch.zeros((1, change.get("rows", 4)), dtype=change.get("positions", torch.int32), device="cuda")
    with pytest.raises(RuntimeError, match=message):
        flash_moba.flash_moba_rotary_func(q, k, pos, change.get("sections"), base=change.get("base", 10000.0), rotary_dim=change.get("rotary_dim"))


def test_the_entry_point_refuses_without_a_gpu():
    import ctypes

    from flash_moba import flash_moba_hip as H

    lib = H.load_library()

    def args(**kw):
        a = H.RotaryArgs()
        a.total, a.heads, a.heads_k, a.head_dim, a.rotary_dim, a.axes, a.log2_base, a.dtype = 16, 4, 2, 64, 64, 1, 13.0, 1
        a.sections[0] = 32
        a.q = a.k = a.q_out = a.k_out = a.positions = 4096
        for name, v in kw.items():
            if name == "section":
                a.sections[0] = v
            else:
                setattr(a, name, v)
        return a

    assert lib.fmoba_rotary(None, None) != 0
    for kw, message in [(dict(dtype=2), b"fp16 and bf16"), (dict(total=-1), b"tokens"), (dict(heads=0, heads_k=0), b"heads"), (dict(head_dim=12), b"head_size"),
                        (dict(rotary_dim=128), b"rotary_dim"), (dict(rotary_dim=4), b"rotary_dim"), (dict(axes=0), b"axes"), (dict(axes=5), b"axes"), (dict(section=31), b"pairs"),
                        (dict(section=-1), b"negative"), (dict(log2_base=-1.0), b"base"), (dict(log2_base=math.nan), b"base"), (dict(q=0), b"null"), (dict(positions=0), b"null"),
                        (dict(q_row_stride=4), b"strides"), (dict(k=4100), b"aligned"), (dict(total=2 ** 31 - 1), b"launch grid")]:
        assert lib.fmoba_rotary(ctypes.byref(args(**kw)), None) != 0, kw
        assert message in lib.fmoba_last_error(), (kw, lib.fmoba_last_error())
    assert lib.fmoba_rotary(ctypes.byref(args(total=0, q=0)), None) == 0  # no tokens: nothing to do
