"""Short norm passes with gradients: not behind the same gradients from elementary torch operations, and nodes of torch's graph
as torch's own are."""
import time

import pytest
import torch
import torch.autograd.forward_ad as fw

from tests.block_util import rand

pytestmark = pytest.mark.gpu
B, S = torch.bfloat16, torch.float32
EPS = 1e-6


@pytest.fixture(scope="module")
def M():
    from bigrig_amd import lib, norm
    lib.init(0)
    return norm


def back(n, s, g):
    return s * (g - n * (g * n).mean(-1, keepdim=True))


def plain_enter(x, w, d):
    """The norm and its gradients in fp32, each result rounded once."""
    v, w32 = x.float(), w.float()
    s = torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
    n = v * s
    d32 = d.float()
    return (n * w32).to(x.dtype), back(n, s, d32 * w32).to(x.dtype), (d32 * n).sum(0).to(w.dtype)


def plain_leave(y, r, gate, nxt, d_new, d_h):
    y32, g32 = y.float(), gate.float()
    new = (r.float() + 0.5 * g32 * y32).to(r.dtype)
    D = d_new.float()
    res = [new]
    if nxt is not None:
        v = new.float()
        s = torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
        n, dh = v * s, d_h.float()
        res.append((n * nxt.float()).to(y.dtype))
        D = D + back(n, s, dh * nxt.float())
    res += [(0.5 * g32 * D).to(y.dtype), D.to(r.dtype), (0.5 * y32 * D).sum(0).to(gate.dtype)]
    if nxt is not None:
        res.append((dh * n).sum(0).to(nxt.dtype))
    return res


def of_a_pass(f, passes=200):
    f()
    torch.cuda.synchronize()
    t = time.perf_counter()
    for _ in range(passes):
        f()
    torch.cuda.synchronize()
    return (time.perf_counter() - t) / passes


def cases(M):
    for T, H, dtype in ((701, 1216, S), (12, 400, B)):
        x, w, d = rand((T, H), dtype, 1).requires_grad_(), rand((H,), dtype, 2).requires_grad_(), rand((T, H), dtype, 3)

        def own(x=x, w=w, d=d):
            return torch.autograd.grad(M.enter(x, w, EPS), (x, w), d)

        yield f"enter {T} x {H} {dtype}", own, lambda x=x, w=w, d=d: plain_enter(x.detach(), w.detach(), d)
    for T, H, dtype, nxt in ((699, 1856, B, False), (56, 1920, S, True)):
        y, r = (rand((T, H), dtype, i).requires_grad_() for i in (1, 2))
        g, n = (rand((H,), dtype, i).requires_grad_() for i in (3, 4))
        d = [rand((T, H), dtype, i) for i in (5, 6)]
        n = n if nxt else None

        def own(y=y, r=r, g=g, n=n, d=d):
            out = M.leave(y, r, None, g, 0.5, n, EPS)
            return torch.autograd.grad(out, [t for t in (y, r, g, n) if t is not None], d if n is not None else d[0])

        yield (f"leave {T} x {H} {dtype}", own,
               lambda y=y, r=r, g=g, n=n, d=d: plain_leave(y.detach(), r.detach(), g.detach(), n if n is None else n.detach(), *d))


def test_not_behind_torch_operations(M):
    # Blocks in turn, the least of each: what else runs on the machine only adds to a block. (A quarter for the wake-up of torch's
    # thread, 10 or 30 us from one minute to the next.)
    for what, own, plain in cases(M):
        a, b = (min(v) for v in zip(*((of_a_pass(own), of_a_pass(plain)) for _ in range(7))))
        assert a < 1.25 * b, f"{what}: {a * 1e6:.1f} us, of torch's operations {b * 1e6:.1f}"


def test_no_python_in_a_gradient(M):
    # a node written in Python takes the interpreter on the thread that runs gradients
    x, w = rand((5, 72), S, 1).requires_grad_(), rand((72,), S, 2)
    for out in (M.enter(x), M.enter(x, w), M.leave(x, x), *M.leave(x, x, w, w, 1.0, w)):
        assert out.grad_fn.name() == "BlockNormBackward" and not isinstance(out.grad_fn, torch.autograd.function.BackwardCFunction)


def test_released_changed_and_kept_graphs(M):
    x, w = rand((5, 72), S, 1).requires_grad_(), rand((72,), S, 2).requires_grad_()
    r = rand((5, 72), S, 3)
    for make in (lambda: M.enter(x, w), lambda: M.leave(x, r, w, None, 1.0, w)[1], lambda: M.leave(x, r, w)):
        h = make()
        a = torch.autograd.grad(h.sum(), (x, w), retain_graph=True)
        b = torch.autograd.grad(h.sum(), (x, w))
        assert all(torch.equal(p, q) for p, q in zip(a, b))
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(h.sum(), (x, w))
        h = make()
        with torch.no_grad():
            w.mul_(1.0)
        with pytest.raises(RuntimeError, match="inplace"):
            torch.autograd.grad(h.sum(), (x, w))
    # what a caller's hooks do to saved tensors is done to these, too
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (seen.append(1), t.cpu())[1], lambda t: t.cuda()):
        h = M.leave(x, r, w, None, 1.0, w)[1]
    assert len(seen) >= 4 and all(torch.isfinite(t).all() for t in torch.autograd.grad(h.sum(), (x, w)))
    # leaves' gradients add up, through a result used twice
    x.grad = None
    h = M.enter(x, w)
    (h + 2 * h).sum().backward(inputs=[x])
    (one,) = torch.autograd.grad(M.enter(x, w), x, torch.full((5, 72), 3.0, device="cuda"))
    assert torch.equal(x.grad, one)


def test_a_gradient_with_a_tangent_is_refused(M):
    x = rand((4, 8), S, 1).requires_grad_()
    with fw.dual_level():
        h = M.enter(x)
        with pytest.raises(RuntimeError, match="tangent"):
            torch.autograd.grad(h, x, fw.make_dual(torch.ones_like(h), torch.ones_like(h)))


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_in_a_compiled_function(M, backend):
    # (torch's graph breaks at the calls)
    ts = [rand((5, 72), S, 1), rand((72,), S, 2), rand((5, 72), S, 3)]

    def block(x, w, r):
        new, h = M.leave(M.enter(x, w) * 2, r, w, None, 0.5, w)
        return new + h

    for grad in (False, True):
        torch._dynamo.reset()
        a, b = ([t.clone().requires_grad_(grad) for t in ts] for _ in range(2))
        got, want = torch.compile(block, backend=backend)(*a), block(*b)
        assert torch.equal(got, want) and got.requires_grad == grad
        if grad:
            d = rand((5, 72), S, 4)
            assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(got, a, d), torch.autograd.grad(want, b, d)))


def test_transforms_without_a_rule_are_refused(M):
    x, w = rand((5, 72), S, 1), rand((72,), S, 2)
    for f in (lambda v: M.enter(v, w).sum(), lambda v: M.leave(v, v, w, None, 1.0, w)[1].sum()):
        for call in (lambda: torch.func.grad(f)(x), lambda: torch.func.jvp(f, (x,), (x,)), lambda: torch.func.vmap(f)(x[None])):
            with pytest.raises(RuntimeError):
                call()


def test_the_residuals_gradient_without_a_next_norm(M):
    # is the one given, whichever others are asked for
    y, r, w = rand((30, 264), B, 1), rand((30, 264), S, 2), rand((264,), B, 3)
    for d in (rand((30, 264), S, 4), rand((264, 30), S, 5).t(), torch.ones((1, 1), device="cuda").expand(30, 264)):
        for needs in ((0, 1, 0), (1, 1, 0), (0, 1, 1), (1, 1, 1), (1, 0, 1)):
            ts = [t.clone().requires_grad_(bool(n)) for t, n in zip((y, r, w), needs)]
            asked = [t for t, n in zip(ts, needs) if n]
            got = torch.autograd.grad(M.leave(*ts), asked, d)
            whole = [t.clone().requires_grad_() for t in (y, r, w)]
            want = torch.autograd.grad(M.leave(*whole), whole, d.clone())
            assert all(torch.equal(a, b) for a, b in zip(got, (v for v, n in zip(want, needs) if n)))
            if needs[1]:
                assert torch.equal(got[needs[0]], d)
    # added to what is there, it leaves the gradient that was given as it was
    r2, d = r.clone().requires_grad_(), rand((30, 264), S, 6)
    keep = d.clone()
    for _ in range(2):
        M.leave(y, r2).backward(d)
    assert torch.equal(d, keep) and torch.equal(r2.grad, 2 * keep)
