"""The transformer-block operators of torch_ops (RMS norm with residual and 8-bit output, row quantisation, rotary positions, linear with
activation and residual in 16 and 8 bits) against plain implementations in 64 bits.

Tolerances.  A result rounded to type t is off by at most half a step, finfo(t).eps / 2 of its value (e4m3: 2^-4).  The f32 arithmetic in
front of that rounding adds, for a sum of n terms accumulated in any order, at most (n + c) 2^-24 of the sum of the terms' magnitudes;
what a matrix product's blocked accumulation really does is far below n 2^-24, so `F32 = 2^-19` of the magnitudes (32 roundings in a row)
is what the tests allow, and they compute those magnitudes."""
import math

import pytest
import torch

F32 = 2.0 ** -19
HALF = [torch.bfloat16, torch.float16]


def T():
    import miphei_vit_amd.torch_ops as ops
    return ops


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


# 16-bit outputs of e4m3 products come from instructions that add neighbouring products with 13 bits below the largest of them: each
# product is off by at most 2^-13 of a product of its group, the sum by at most 2^-13 of the groups' largest, which is below the magnitudes
F8 = 2.0 ** -13


def close(got, want, mag, what="", f32=F32):
    """got (rounded to its type) against want (f64); mag: magnitudes of what was summed (f64)"""
    t = got.dtype
    tiny = torch.finfo(t).smallest_normal * torch.finfo(t).eps if t != torch.float32 else 1e-37
    tol = torch.finfo(t).eps / 2 * want.abs() + f32 * mag + tiny
    err = (got.double() - want).abs()
    worst = (err - tol).max().item() if err.numel() else -1.0
    assert not err.numel() or bool((err <= tol).all()), f"{what}: over by {worst:.3e} at {int((err - tol).argmax())}, max err {err.max().item():.3e}"


def e4m3_round(v):
    """v (f64) to the nearest e4m3 value, ties to even"""
    _, e = torch.frexp(v)
    step = torch.exp2((e - 1).clamp_min(-6).double() - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


# ------------------------------------------------------------------ registration and refusals (no GPU needed)
NAMES = ("rms_norm_forward", "rms_norm_backward", "rms_norm_fp8", "quantize_fp8", "rotary_forward", "rotary_", "linear_act_forward",
         "linear_act_backward", "linear_fp8")


def test_registered_without_cpu_kernels():
    ops = T()
    for name in NAMES:
        assert hasattr(torch.ops.mvit, name), name
    x = torch.zeros(2, 16)
    with pytest.raises(NotImplementedError):
        ops.rms_norm(x, torch.ones(16))
    with pytest.raises(NotImplementedError):
        ops.quantize_fp8(x)


def fake(*shape, dtype=torch.bfloat16, device="cuda"):
    return torch.empty(*shape, dtype=dtype, device=device)


def test_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops = T()
    f32, f8 = torch.float32, torch.float8_e4m3fn
    with FakeTensorMode():
        x, r, w = fake(2, 5, 48), fake(2, 5, 48, dtype=f32), fake(48, dtype=f32)
        y, h = ops.add_rms_norm(x, r, w)
        assert y.dtype == torch.bfloat16 and h.dtype == f32 and y.shape == h.shape == x.shape
        assert ops.rms_norm(r, w, out_dtype=torch.float16).dtype == torch.float16
        q, s, h = ops.add_rms_norm_fp8(x, x, w)
        assert q.dtype == f8 and s.shape == (2, 5) and s.dtype == f32 and h.dtype == torch.bfloat16
        q, s = ops.quantize_fp8(x)
        assert q.shape == x.shape and q.dtype == f8
        z = ops.rotary(fake(2, 7, 6, 16), fake(6, 2, dtype=torch.int32), fake(8, dtype=f32), [4, 4], 4, 1)
        assert z.shape == (2, 7, 6, 16)
        wt = fake(24, 48)
        assert ops.linear_act(x, wt, fake(24), None, "gelu").dtype == torch.bfloat16
        assert ops.linear_act(x, wt, None, fake(2, 5, 24, dtype=f32)).dtype == f32
        assert ops.linear_fp8(q, s, fake(24, 48, dtype=f8), fake(24, dtype=f32), out_dtype=f32).shape == (2, 5, 24)


def refusals():
    f32, f16, f8, i32 = torch.float32, torch.float16, torch.float8_e4m3fn, torch.int32
    x, w = fake(4, 48), fake(48, dtype=f32)
    p, fr = fake(7, 2, dtype=i32), fake(8, dtype=f32)
    rx = fake(2, 7, 6, 16)
    lw, s = fake(24, 48), fake(4, dtype=f32)
    q8, w8, ws = fake(4, 48, dtype=f8), fake(24, 48, dtype=f8), fake(24, dtype=f32)
    return {
        "norm weight": lambda o: o.rms_norm(x, fake(47, dtype=f32)),
        "norm residual broadcast": lambda o: o.add_rms_norm(x, fake(1, 48), w),
        "norm mixed halves": lambda o: o.add_rms_norm(x, fake(4, 48, dtype=f16), w),
        "norm f32 with half residual": lambda o: o.add_rms_norm(fake(4, 48, dtype=f32), x, w),
        "norm f64": lambda o: o.rms_norm(fake(4, 48, dtype=torch.float64), w),
        "norm integers": lambda o: o.rms_norm(fake(4, 48, dtype=i32), w),
        "norm out dtype": lambda o: o.rms_norm(x, w, 1e-6, f32),
        "norm empty rows": lambda o: o.rms_norm(fake(4, 0), fake(0)),
        "norm wide": lambda o: o.rms_norm(fake(4, 16385), fake(16385)),
        "norm scalar": lambda o: o.rms_norm(fake(()), w),
        "norm8 weight": lambda o: o.rms_norm_fp8(x, fake(47, dtype=f32)),
        "quantise wide": lambda o: o.quantize_fp8(fake(4, 16385)),
        "quantise integers": lambda o: o.quantize_fp8(fake(4, 8, dtype=i32)),
        "rotary 3-d": lambda o: o.rotary(fake(7, 6, 16), p, fr, [4, 4]),
        "rotary odd head": lambda o: o.rotary(fake(2, 7, 6, 15), p, fr, [4, 4]),
        "rotary sections": lambda o: o.rotary(rx, p, fr, [4, 5]),
        "rotary no sections": lambda o: o.rotary(rx, p, fr, []) if False else o.rotary(rx, p, fr, [0, 0]),
        "rotary five axes": lambda o: o.rotary(rx, fake(7, 5, dtype=i32), fr, [2, 2, 2, 1, 1]),
        "rotary heads": lambda o: o.rotary(rx, p, fr, [4, 4], 7),
        "rotary prefix": lambda o: o.rotary(rx, p, fr, [4, 4], 6, 8),
        "rotary positions": lambda o: o.rotary(rx, fake(6, 2, dtype=i32), fr, [4, 4]),
        "rotary positions type": lambda o: o.rotary(rx, fake(7, 2, dtype=torch.int16), fr, [4, 4]),
        "rotary frequencies": lambda o: o.rotary(rx, p, fake(7, dtype=f32), [4, 4]),
        "rotary_ expanded": lambda o: torch.ops.mvit.rotary_(rx, p, fr, [4, 4], 7, 0, False),
        "linear K": lambda o: o.linear_act(fake(4, 44), fake(24, 44)),
        "linear weight": lambda o: o.linear_act(x, fake(24, 40)),
        "linear types": lambda o: o.linear_act(x, fake(24, 48, dtype=f16)),
        "linear f32": lambda o: o.linear_act(fake(4, 48, dtype=f32), fake(24, 48, dtype=f32)),
        "linear bias": lambda o: o.linear_act(x, lw, fake(23)),
        "linear residual broadcast": lambda o: o.linear_act(x, lw, None, fake(1, 24)),
        "linear activation": lambda o: o.linear_act(x, lw, None, None, "swish"),
        "linear no columns": lambda o: o.linear_act(x, fake(0, 48)),
        "fp8 types": lambda o: o.linear_fp8(x, s, w8, ws),
        "fp8 K": lambda o: o.linear_fp8(fake(4, 40, dtype=f8), s, fake(24, 40, dtype=f8), ws),
        "fp8 scale": lambda o: o.linear_fp8(q8, fake(3, dtype=f32), w8, ws),
        "fp8 scale type": lambda o: o.linear_fp8(q8, fake(4), w8, ws),
        "fp8 out type": lambda o: o.linear_fp8(q8, s, w8, ws, out_dtype=torch.float64),
    }


@pytest.mark.parametrize("name", ["norm weight", "norm residual broadcast", "norm mixed halves", "norm f32 with half residual", "norm f64",
                                  "norm integers", "norm out dtype", "norm empty rows", "norm wide", "norm scalar", "norm8 weight",
                                  "quantise wide", "quantise integers", "rotary 3-d", "rotary odd head", "rotary sections", "rotary no sections",
                                  "rotary five axes", "rotary heads", "rotary prefix", "rotary positions", "rotary positions type",
                                  "rotary frequencies", "rotary_ expanded", "linear K", "linear weight", "linear types", "linear f32",
                                  "linear bias", "linear residual broadcast", "linear activation", "linear no columns", "fp8 types", "fp8 K",
                                  "fp8 scale", "fp8 scale type", "fp8 out type"])
def test_refused(name):
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        with pytest.raises(ValueError, match="mvit::"):
            refusals()[name](T())


@pytest.mark.gpu
def test_refused_on_two_devices():
    ops = T()
    x = torch.zeros(4, 48, device="cuda", dtype=torch.bfloat16)
    q, s = ops.quantize_fp8(x)
    for call in (lambda: ops.rms_norm(x, torch.ones(48)), lambda: ops.add_rms_norm(x, x.cpu(), torch.ones(48, device="cuda")),
                 lambda: ops.rotary(x.view(1, 4, 3, 16), torch.zeros(4, 1, dtype=torch.int32), torch.ones(8, device="cuda"), [8]),
                 lambda: ops.linear_act(x, torch.zeros(8, 48, dtype=torch.bfloat16)), lambda: ops.linear_fp8(q, s.cpu(), q, s)):
        with pytest.raises(ValueError, match="mvit::"):
            call()


def test_c_entries_refuse_what_they_cannot_do():
    """the C-ABI by itself: bad sizes, types and strides come back as -1 before anything is launched (addresses are never read here)"""
    import ctypes as C
    from miphei_vit_amd import _lib as L
    lib, p = L.lib(), 4096
    norm = lambda M, D, ldx=None, x_f32=0, res=None, res_f32=0, y_f32=0: lib.mvit_rmsnorm_fwd(  # noqa: E731
        p, x_f32, D if ldx is None else ldx, res, res_f32, D, p, 1, p, p, y_f32, None, M, D, 1e-6, None)
    assert norm(-1, 8) == norm(4, 0) == norm(4, 16385) == norm(4, 8, ldx=7) == norm(4, 8, y_f32=1) == norm(4, 8, x_f32=1, res=p) == -1
    assert lib.mvit_rmsnorm_fwd(None, 0, 8, None, 0, 0, p, 1, None, p, 0, None, 4, 8, 1e-6, None) == -1
    assert norm(0, 8) == 0
    assert lib.mvit_quantize_rows_fp8(p, 0, 8, p, None, 4, 8, None) == -1
    assert lib.mvit_rmsnorm_bwd(p, 0, None, p, 0, p, 1, p, p, None, p, None, 0, 4, 8, None) == -1          # dw without scratch
    a = L.RotaryArgs(x=p, y=p, positions=p, inv_freq=p, B=1, N=2, H=2, Dh=8, rotate_heads=2, axes=1)
    a.sections[0] = 4

    def rot(**kw):
        b = L.RotaryArgs.from_buffer_copy(a)
        for k, v in kw.items():
            if k == "sections":
                b.sections[0] = v
            else:
                setattr(b, k, v)
        return lib.mvit_rotary(C.byref(b), None)
    assert all(rot(**kw) == -1 for kw in (dict(Dh=7), dict(Dh=1026), dict(H=1025), dict(rotate_heads=3), dict(prefix=3), dict(axes=0), dict(axes=5),
                                          dict(sections=5), dict(sections=0), dict(sections=-1), dict(pos_type=3), dict(x=None), dict(B=-1)))
    assert rot(N=0) == rot(B=0) == 0
    a = L.LinearArgs(x=p, w=p, y=p, x_scale=p, w_scale=p, ldx=16, ldw=16, M=4, N=4, K=16)

    def lin(fn, **kw):
        b = L.LinearArgs.from_buffer_copy(a)
        for k, v in kw.items():
            setattr(b, k, v)
        return fn(C.byref(b), None)
    for fn in (lib.mvit_linear_act, lib.mvit_linear_fp8):
        assert all(lin(fn, **kw) == -1 for kw in (dict(K=12), dict(K=0), dict(N=0), dict(M=-1), dict(ldx=8), dict(ldx=20), dict(ldw=17), dict(act=5),
                                                  dict(act=-1), dict(x=p + 8), dict(w=p + 2), dict(y=None), dict(res=p, ldr=3), dict(ldx=1 << 24)))
        assert lin(fn, M=0) == 0
    assert lin(lib.mvit_linear_fp8, pre=p) == lin(lib.mvit_linear_fp8, x_scale=None) == -1
    act = lambda pre=p, dz=p, ldz=8, db=None, s=None: lib.mvit_act_bwd(p, 0, pre, 3, dz, ldz, db, 0, s, 4, 8, None)  # noqa: E731
    assert act(pre=None) == act(db=p) == act(ldz=4) == act(ldz=12) == act(dz=p + 2) == -1
    a = L.LinearArgs(x=p, w=p, y=p, ldx=16, ldw=16, M=4, N=16, K=16)
    for rows in (0, 1):
        grad = lambda **kw: lin(lambda b, s: lib.mvit_linear_grad(b, rows, p, 1 << 40, s), **kw)  # noqa: E731
        assert all(grad(**kw) == -1 for kw in (dict(M=0), dict(N=0), dict(N=12), dict(K=0), dict(ldx=12), dict(ldw=8), dict(ldw=20), dict(x=p + 8), dict(w=p + 2),
                                               dict(y=p + 4), dict(y=None), dict(bias=p), dict(res=p), dict(pre=p), dict(act=1), dict(y_f32=1), dict(ldw=1 << 23)))
        assert grad(ldx=8) == -1 or rows
    assert lib.mvit_linear_grad(C.byref(L.LinearArgs(x=p, w=p, y=p, ldx=8, ldw=16, M=9, N=16, K=4)), 1, None, 0, None) == -1      # 9 columns in rows of 8
    assert lib.mvit_linear_grad_scratch_bytes(64, 512, 20816) > 0 == lib.mvit_linear_grad_scratch_bytes(4, 8, 64)
    assert lib.mvit_linear_grad(C.byref(L.LinearArgs(x=p, w=p, y=p, ldx=64, ldw=512, M=64, N=512, K=20816)), 1, p, 64, None) == -1


def test_frequencies_and_grid():
    ops = T()
    f = ops.rotary_frequencies([2, 3], 100.0)
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1.0, 100 ** -0.5, 1.0, 100 ** (-1 / 3), 100 ** (-2 / 3)], dtype=torch.float64))
    f = ops.rotary_frequencies([2, 2], 16.0, shared=True)
    assert torch.allclose(f, torch.tensor([1.0, 0.5, 0.25, 0.125], dtype=torch.float64))
    assert ops.grid_positions(2, 3).tolist() == [[0, 0], [0, 1], [0, 2], [1, 0], [1, 1], [1, 2]]


# ------------------------------------------------------------------ RMS norm
NORM_TYPES = [(torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.float16, torch.float32),
              (torch.float32, torch.float32), (torch.bfloat16, None), (torch.float32, None)]
# one row; a row of one value; widths at the borders of the layouts, odd ones, ones no piece fits; more rows than the grid has waves
NORM_SIZES = [(1, 1), (3, 7), (1, 1536), (5, 512), (1037, 520), (1100, 1000), (70, 1531), (1030, 2048), (40, 4096), (1030, 4096), (9, 8192),
              (3, 16384), (2, 16383), (17, 4100), (9001, 64)]


def norm_oracle(h, w, eps):
    h, w = h.double(), w.double()
    rstd = (h.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    return h * rstd * w, rstd


@pytest.mark.gpu
@pytest.mark.parametrize("types", NORM_TYPES, ids=lambda t: "-".join(str(v).replace("torch.", "") for v in t))
@pytest.mark.parametrize("M,D", NORM_SIZES)
def test_rms_norm_forward_backward(M, D, types):
    ops, g = T(), gen(M * 31 + D)
    xt, rt = types
    x = randn(g, M, D, dtype=xt).requires_grad_()
    w = (1 + 0.2 * torch.randn(D, device="cuda", generator=g)).to(torch.float32 if M % 2 else xt).requires_grad_()
    r = None if rt is None else randn(g, M, D, dtype=rt, scale=3).requires_grad_()
    if r is None:
        y = ops.rms_norm(x, w, 1e-5)
        h = x.detach()
    else:
        y, h = ops.add_rms_norm(x, r, w, 1e-5)
        hd = x.detach().double() + r.detach().double()
        close(h.detach(), hd, hd.abs(), "h")
        assert h.dtype == rt
    assert y.dtype == xt
    want, rstd = norm_oracle(h.detach(), w.detach(), 1e-5)
    close(y.detach(), want, want.abs(), "y")
    dy = randn(g, M, D, dtype=xt)
    dh = None if r is None else randn(g, M, D, dtype=rt)
    leaves = (x, w) if r is None else (x, r, w)
    grads = torch.autograd.grad((y,) if r is None else (y, h), leaves, (dy,) if r is None else (dy, dh))
    hd, wd, dyd = h.detach().double(), w.detach().double(), dy.double()
    xhat = hd * rstd
    wdy = wd * dyd
    base = torch.zeros_like(hd) if dh is None else dh.double()
    total = base + rstd * (wdy - xhat * (wdy * xhat).mean(-1, keepdim=True))
    mag = base.abs() + rstd * (wdy.abs() + xhat.abs() * (wdy * xhat).abs().mean(-1, keepdim=True))
    close(grads[0], total, mag, "dx")
    if r is not None:
        close(grads[1], total, mag, "dresidual")
    close(grads[-1], (dyd * xhat).sum(0), (dyd * xhat).abs().sum(0), "dweight")
    assert grads[-1].dtype == w.dtype


@pytest.mark.gpu
def test_rms_norm_gradient_against_differences():
    ops, g = T(), gen(3)
    M, D = 3, 40
    x, r, w = (randn(g, *s) for s in ((M, D), (M, D), (D,)))
    cy, ch = randn(g, M, D), randn(g, M, D)
    leaves = [t.clone().requires_grad_() for t in (x, r, w)]
    y, h = ops.add_rms_norm(*leaves, 1e-3)
    grads = torch.autograd.grad((y, h), leaves, (cy, ch))

    def f(x, r, w):
        h = x + r
        return float((norm_oracle(h, w, 1e-3)[0] * cy).sum() + (h * ch).sum())
    step = 1e-5      # central differences of the 64-bit function: O(step^2) and 1e-16 / step away from its derivative
    for which, grad in enumerate(grads):
        for i in (0, 7, grad.numel() - 1):
            args = [t.double().clone() for t in (x, r, w)]
            args[which].view(-1)[i] += step
            up = f(*args)
            args[which].view(-1)[i] -= 2 * step
            d = (up - f(*args)) / (2 * step)
            assert abs(d - float(grad.view(-1)[i])) <= 1e-5 * max(1.0, abs(d)), (which, i)


@pytest.mark.gpu
def test_rms_norm_partial_gradients():
    """y alone, h alone, and each leaf alone"""
    ops, g = T(), gen(4)
    x, r = randn(g, 6, 96, dtype=torch.bfloat16).requires_grad_(), randn(g, 6, 96).requires_grad_()
    w = randn(g, 96).requires_grad_()
    dy, dh = randn(g, 6, 96, dtype=torch.bfloat16), randn(g, 6, 96)
    y, h = ops.add_rms_norm(x, r, w)
    all_y = torch.autograd.grad(y, (x, r, w), dy, retain_graph=True)
    only_h = torch.autograd.grad(h, (x, r, w), dh, retain_graph=True, materialize_grads=True)
    assert torch.equal(only_h[0], dh.to(torch.bfloat16)) and torch.equal(only_h[1], dh) and not only_h[2].any()
    for k, leaf in enumerate((x, r, w)):
        other = [t.detach().clone().requires_grad_(j == k) for j, t in enumerate((x, r, w))]
        y1, _ = ops.add_rms_norm(*other)
        assert torch.equal(torch.autograd.grad(y1, other[k], dy)[0], all_y[k])


@pytest.mark.gpu
def test_rms_norm_types_strides_empty():
    ops, g = T(), gen(5)
    w = randn(g, 64)
    stream = randn(g, 4, 64)
    y = ops.rms_norm(stream, w, out_dtype=torch.float16)
    close(y, norm_oracle(stream, w, 1e-6)[0], norm_oracle(stream, w, 1e-6)[0].abs())
    big = randn(g, 6, 3, 200, dtype=torch.bfloat16)
    for view in (big[:, 1, 8:72], big[:, 1, 3:67], big[::2, :, 8:72], big[:, :, 8:72].transpose(0, 1), big[0, 0, :64].expand(5, 64)):
        got = ops.rms_norm(view, w)
        assert torch.equal(got, ops.rms_norm(view.contiguous(), w)) and got.shape == view.shape
        y, h = ops.add_rms_norm(view, view, w)
        y2, h2 = ops.add_rms_norm(view.contiguous(), view.contiguous(), w)
        assert torch.equal(y, y2) and torch.equal(h, h2)
    e = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    wg = w.clone().requires_grad_()
    y, h = ops.add_rms_norm(e, torch.empty(0, 64, device="cuda"), wg)
    de, dw = torch.autograd.grad(y.float().sum() + h.sum(), (e, wg))
    assert y.shape == h.shape == de.shape == (0, 64) and not dw.any()
    q, s = ops.rms_norm_fp8(e.detach(), w)
    assert q.shape == (0, 64) and s.shape == (0,)


@pytest.mark.gpu
def test_rms_norm_is_the_same_every_time():
    ops, g = T(), gen(6)
    x, r, w = randn(g, 5000, 384, dtype=torch.bfloat16).requires_grad_(), randn(g, 5000, 384).requires_grad_(), randn(g, 384).requires_grad_()
    dy, dh = randn(g, 5000, 384, dtype=torch.bfloat16), randn(g, 5000, 384)
    runs = []
    for _ in range(3):
        y, h = ops.add_rms_norm(x, r, w)
        runs.append((y, h, *torch.autograd.grad((y, h), (x, r, w), (dy, dh))))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


# ------------------------------------------------------------------ 8 bits
def check_e4m3(q, scale, y, mag=None):
    """q * scale is y rounded: half an e4m3 step of y / scale (2^-4 of it; 2^-10 below the smallest normal, 2^-6), and f32 in front of it"""
    amax = y.abs().amax(-1)
    want = amax.clamp_min(1e-30) / 448
    assert torch.allclose(scale.double(), want, rtol=2 ** -18, atol=0)
    s = scale.double()[..., None]
    tol = torch.maximum(y.abs() * 2.0 ** -4, s * 2.0 ** -10) + F32 * (y.abs() if mag is None else mag)
    assert bool(((q.double() * s - y).abs() <= tol).all())


@pytest.mark.gpu
@pytest.mark.parametrize("types", [t for t in NORM_TYPES], ids=lambda t: "-".join(str(v).replace("torch.", "") for v in t))
@pytest.mark.parametrize("M,D", NORM_SIZES)
def test_rms_norm_fp8(M, D, types):
    ops, g = T(), gen(M * 17 + D)
    xt, rt = types
    x, w = randn(g, M, D, dtype=xt), 1 + 0.2 * randn(g, D)
    if rt is None:
        q, scale = ops.rms_norm_fp8(x, w, 1e-5)
        h = x
    else:
        r = randn(g, M, D, dtype=rt, scale=3)
        q, scale, h = ops.add_rms_norm_fp8(x, r, w, 1e-5)
        assert torch.equal(h, ops.add_rms_norm(x, r, w, 1e-5)[1])
    check_e4m3(q, scale, norm_oracle(h, w, 1e-5)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,D", NORM_SIZES)
def test_quantize_fp8(M, D, dtype):
    ops, g = T(), gen(M * 7 + D)
    x = randn(g, M, D, dtype=dtype, scale=5)
    x[M // 2] = 0                                    # a row of nothing
    q, scale = ops.quantize_fp8(x)
    check_e4m3(q, scale, x.double())
    assert not q[M // 2].float().any()
    # to the last bit: x / scale in f32, rounded to nearest even (ties, which a 16-bit row is full of, included)
    want = (x.float() / scale[:, None]).to(torch.float64)
    assert torch.equal(q.double(), e4m3_round(want))


@pytest.mark.gpu
def test_non_finite_rows_read_back_as_nan_and_stay_alone():
    ops, g = T(), gen(9)
    x = randn(g, 6, 96, dtype=torch.bfloat16)
    clean_q, clean_s = ops.quantize_fp8(x)
    x[1, 5] = float("nan")
    x[3, 95] = float("inf")
    x[4, 0] = float("-inf")
    q, s = ops.quantize_fp8(x)
    back = q.float() * s[:, None]
    for row in (1, 3, 4):
        assert back[row].isnan().all()
    for row in (0, 2, 5):
        assert torch.equal(q[row].float(), clean_q[row].float()) and s[row] == clean_s[row]
    w = torch.ones(96, device="cuda")
    y = ops.rms_norm(x, w)
    q, s = ops.rms_norm_fp8(x, w)
    back = q.float() * s[:, None]
    for row in (1, 3, 4):
        assert y[row].isnan().any() and back[row].isnan().all()
    for row in (0, 2, 5):
        assert y[row].isfinite().all() and back[row].isfinite().all()
    low = torch.full((2, 96), torch.finfo(torch.bfloat16).min, device="cuda", dtype=torch.bfloat16)   # the type's lowest value
    q, s = ops.quantize_fp8(low)
    assert (q.float() == -448).all() and torch.allclose(q.float() * s[:, None], low.float())
    tiny = torch.full((1, 96), 1e-38, device="cuda")
    q, s = ops.quantize_fp8(tiny)
    assert s.isfinite().all() and (s > 0).all() and q.float().isfinite().all()


@pytest.mark.gpu
def test_no_gradient_where_there_is_none():
    ops = T()
    x = torch.randn(4, 32, device="cuda", requires_grad=True)
    w = torch.ones(32, device="cuda")
    for call in (lambda: ops.quantize_fp8(x), lambda: ops.rms_norm_fp8(x, w), lambda: ops.add_rms_norm_fp8(x.detach(), x, w)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
        with torch.no_grad():
            call()


# ------------------------------------------------------------------ rotary
def rotary_oracle(x, pos, freq, sections, rot, prefix, interleaved, sign=1):
    """(result, magnitudes) in f64"""
    P = sum(sections)
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], device=x.device)
    x = x.double()
    out, mag = x.clone(), x.abs()
    angle = pos.double()[..., axis] * freq.double()
    c, s = angle.cos().unsqueeze(-2), sign * angle.sin().unsqueeze(-2)
    i = torch.arange(P, device=x.device)
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + P)
    v = x[:, prefix:, :rot]
    a, b = v[..., ia], v[..., ib]
    out[:, prefix:, :rot, ia.tolist()] = a * c - b * s
    out[:, prefix:, :rot, ib.tolist()] = b * c + a * s
    both = a.abs() + b.abs()
    mag[:, prefix:, :rot, ia.tolist()] = both
    mag[:, prefix:, :rot, ib.tolist()] = both
    return out, mag


ROTARY = [  # B, N, heads, head_dim, rotated heads, sections, prefix
    (1, 1, 1, 2, 1, [1], 0), (2, 7, 6, 16, 4, [4, 4], 1), (1, 329, 72, 64, 48, [16, 16], 5), (3, 5, 3, 40, 3, [7, 6, 7], 0),
    (2, 9, 4, 128, 4, [16, 24, 24], 0), (1, 6, 5, 48, 2, [3, 5, 2, 1], 2), (2, 3, 2, 256, 2, [128], 0), (1, 5, 9, 32, 0, [16], 0),
    (2, 4, 3, 64, 3, [0, 16], 4), (1, 33, 2, 1024, 1, [200, 300], 1), (2, 5, 3, 80, 2, [20, 20], 0), (1, 2, 2, 12, 2, [3], 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("case", ROTARY, ids=str)
def test_rotary_forward_backward(case, dtype, interleaved):
    ops, g = T(), gen(sum(case[:5]))
    B, N, H, Dh, rot, sections, prefix = case
    x = randn(g, B, N, H, Dh, dtype=dtype).requires_grad_()
    freq = ops.rotary_frequencies(sections, 100.0, device="cuda")
    pos = torch.randint(0, 60, (B, N - prefix, len(sections)), device="cuda", generator=g)
    y = ops.rotary(x, pos, freq, sections, rot, prefix, interleaved)
    want, mag = rotary_oracle(x.detach(), pos, freq, sections, rot, prefix, interleaved)
    close(y.detach(), want, mag, "y")
    same = (want == x.detach().double()) & (mag == want.abs())      # what passes through, to the bit
    assert torch.equal(y.detach()[same], x.detach()[same])
    dy = randn(g, B, N, H, Dh, dtype=dtype)
    (dx,) = torch.autograd.grad(y, x, dy)
    close(dx, *rotary_oracle(dy, pos, freq, sections, rot, prefix, interleaved, -1), "dx")
    z = x.detach().clone()
    assert ops.rotary_(z, pos, freq, sections, rot, prefix, interleaved) is z
    assert torch.equal(z, y.detach())


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_layouts_and_positions(interleaved):
    ops, g = T(), gen(11)
    B, N, H, Dh, sections = 2, 13, 4, 32, [6, 10]
    freq = ops.rotary_frequencies(sections, 100.0, device="cuda")
    pos = torch.randint(-20, 20, (N, 2), device="cuda", generator=g, dtype=torch.int32)
    x = randn(g, B, N, H, Dh, dtype=torch.bfloat16)
    want = ops.rotary(x, pos, freq, sections, interleaved=interleaved)
    heads = x.transpose(1, 2).contiguous().transpose(1, 2)                        # head-major
    got = ops.rotary(heads, pos, freq, sections, interleaved=interleaved)
    assert torch.equal(got, want) and got.stride() == heads.stride()
    packed = randn(g, B, N, 3 * H + 1, Dh, dtype=torch.bfloat16)                  # a slice of a wider projection, one value off 16 bytes
    packed[:, :, 1:1 + H] = x
    assert torch.equal(ops.rotary(packed[:, :, 1:1 + H], pos, freq, sections, interleaved=interleaved), want)
    odd = torch.zeros(B * N * H * Dh + 1, device="cuda", dtype=torch.bfloat16)[1:].view(B, N, H, Dh).copy_(x)
    assert torch.equal(ops.rotary(odd, pos, freq, sections, interleaved=interleaved), want)
    last = x.transpose(2, 3).contiguous().transpose(2, 3)                         # head_dim not the last in memory
    assert torch.equal(ops.rotary(last, pos, freq, sections, interleaved=interleaved), want)
    for p in (pos.long(), pos.float(), pos.expand(B, N, 2), pos.t().contiguous().t()):
        assert torch.equal(ops.rotary(x, p, freq, sections, interleaved=interleaved), want)
    y = ops.rotary(x, pos, freq.float(), sections, interleaved=interleaved)       # f32 frequencies: other angles, the same formula
    close(y, *rotary_oracle(x, pos, freq.float(), sections, H, 0, interleaved))
    w = packed.clone()
    ops.rotary_(w[:, :, 1:1 + H], pos, freq, sections, interleaved=interleaved)   # in place in a slice: the rest is left alone
    assert torch.equal(w[:, :, 1:1 + H], want) and torch.equal(w[:, :, :1], packed[:, :, :1]) and torch.equal(w[:, :, 1 + H:], packed[:, :, 1 + H:])
    with pytest.raises(ValueError, match="in place"):
        ops.rotary_(last, pos, freq, sections)
    with pytest.raises(ValueError, match="in place"):
        ops.rotary_(x[:, :, :1].expand(B, N, H, Dh), pos, freq, sections)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.rotary_(x.clone().requires_grad_(), pos, freq, sections)
    e = torch.empty(B, 0, H, Dh, device="cuda", requires_grad=True)
    assert ops.rotary(e, pos[:0], freq, sections).shape == (B, 0, H, Dh)


@pytest.mark.gpu
def test_rotary_far_positions_and_gradient_of_gradient():
    ops, g = T(), gen(12)
    freq = ops.rotary_frequencies([32], 10000.0, device="cuda")
    pos = torch.tensor([[2 ** 31 + 12345], [10 ** 9 + 7], [131071], [2 ** 24 + 1]], device="cuda")   # (an f32 angle would be off by whole turns)
    x = randn(g, 1, 4, 2, 64)
    close(ops.rotary(x, pos, freq, [32]), *rotary_oracle(x, pos, freq, [32], 2, 0, False))
    a = randn(g, 1, 4, 2, 64).requires_grad_()
    y = ops.rotary(x.requires_grad_(), pos, freq, [32])
    (dx,) = torch.autograd.grad(y, x, a, create_graph=True)
    (da,) = torch.autograd.grad(dx, a, x.detach())          # the turn back's gradient is the turn
    assert torch.equal(da, y.detach())


@pytest.mark.gpu
def test_rotary_long_offsets():
    """an element offset behind 2^31: 2^21 + 2 tokens of 1024 values, in place in the last ones"""
    ops = T()
    N = 2 ** 21 + 2
    x = torch.zeros(1, N, 16, 64, device="cuda", dtype=torch.bfloat16)
    x[:, -2:] = 1
    freq = ops.rotary_frequencies([32], device="cuda")
    pos = torch.zeros(N, 1, device="cuda", dtype=torch.int32)
    pos[-1] = 3
    ops.rotary_(x, pos, freq, [32])
    assert (x[:, -2] == 1).all() and not x[:, :-2].any()
    one = torch.ones(1, 1, 16, 64, device="cuda", dtype=torch.bfloat16)
    assert torch.equal(x[:, -1:], ops.rotary(one, pos[-1:], freq, [32]))


# ------------------------------------------------------------------ linear
ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh"]


def act_oracle(z, act):
    if act == "relu":
        return z.clamp_min(0), (z > 0).double()
    if act == "silu":
        p = torch.sigmoid(z)
        return z * p, p + z * p * (1 - p)
    if act == "gelu":
        c = torch.special.ndtr(z)
        return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        k = 2 * math.sqrt(2 / math.pi)
        p = torch.sigmoid(k * (z + 0.044715 * z ** 3))
        return z * p, p + z * p * (1 - p) * k * (1 + 3 * 0.044715 * z * z)
    return z, torch.ones_like(z)


# few rows (each of the row kernels), borders of the tiles, ragged everything, K of one piece, columns no store fits
LINEAR = [(1, 8, 1), (1, 1536, 1536), (5, 64, 33), (16, 136, 24), (17, 4096, 130), (32, 200, 72), (33, 96, 288), (64, 64, 64), (65, 72, 129),
          (329, 1536, 200), (1301, 96, 515), (2100, 264, 2056), (3000, 1544, 1100), (4111, 128, 1031),
          # the largest tiles: one a block, ragged and not, several a block (with a K of one and of an odd number of K tiles)
          (5003, 72, 2397), (5000, 512, 2400), (8200, 328, 2600), (12000, 8, 2600),
          # each of the tiles: 64 x 64, 128 x 128, 128 x 256, 192 x 256, 256 x 256, the last two several a block
          (329, 264, 1000), (700, 136, 4096), (1301, 200, 4608), (5264, 136, 4096), (5260, 72, 4093), (5264, 88, 8192), (5300, 40, 8181)]


def linear_case(g, M, K, N, dtype, res, bias_f32):
    x, w = randn(g, M, K, dtype=dtype), randn(g, N, K, dtype=dtype, scale=K ** -0.5)
    b = randn(g, N, dtype=torch.float32 if bias_f32 else dtype)
    r = None if res is None else randn(g, M, N, dtype=res)
    return x, w, b, r


@pytest.mark.gpu
@pytest.mark.parametrize("res", ["none", "half", "f32"])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("M,K,N", LINEAR)
def test_linear_act_forward_backward(M, K, N, dtype, res):
    ops, g = T(), gen(M + K + N)
    act = ACTS[(M + N + len(res)) % 5]
    rt = {"none": None, "half": dtype, "f32": torch.float32}[res]
    x, w, b, r = linear_case(g, M, K, N, dtype, rt, False)
    leaves = [t.requires_grad_() for t in (x, w, b, r) if t is not None]
    y = ops.linear_act(x, w, b, r, act)
    assert y.dtype == (rt or dtype)
    xd, wd, bd = x.detach().double(), w.detach().double(), b.detach().double()
    z = xd @ wd.t() + bd
    zmag = xd.abs() @ wd.abs().t() + bd.abs()
    out, slope = act_oracle(z, act)
    rd = torch.zeros_like(z) if r is None else r.detach().double()
    close(y.detach(), out + rd, 1.2 * zmag + rd.abs(), "y")       # |act'| <= 1.13 for all of them
    dy = randn(g, M, N, dtype=y.dtype)
    grads = torch.autograd.grad(y, leaves, dy)
    # dz is rounded to 16 bits (half a step each), and z is kept in 16 bits: |act''| <= 1 there
    half = torch.finfo(dtype).eps / 2
    dyd = dy.double()
    dz = dyd * slope
    dz_off = dz.abs() * half + (dyd.abs() * z.abs() * half if act not in ("none", "relu") else 0) + F32 * dyd.abs() * (1 + zmag)
    if act == "relu":   # a z within its rounding of 0 may fall on either side
        dz_off = dz_off + dyd.abs() * (z.abs() <= zmag * F32).double()
    tiny = torch.finfo(dtype).smallest_normal

    def grad_close(got, want, off, mag, what):
        tol = torch.finfo(got.dtype).eps / 2 * (want.abs() + off) + off + F32 * mag + tiny
        err = (got.double() - want).abs()
        assert bool((err <= tol).all()), f"{what}: max err {err.max():.3e}, over by {(err - tol).max():.3e}"
    grad_close(grads[0], dz @ wd, dz_off @ wd.abs(), dz.abs() @ wd.abs(), "dx")
    grad_close(grads[1], dz.t() @ xd, dz_off.t() @ xd.abs(), dz.abs().t() @ xd.abs(), "dweight")
    grad_close(grads[2], dz.sum(0), dz_off.sum(0), dz.abs().sum(0), "dbias")
    if r is not None:
        assert torch.equal(grads[3], dy)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTS)
def test_linear_act_gradient_against_differences(act):
    """the activation's slope: dbias of one row and K = 8, f32 dy and bias, against central differences of the 64-bit function"""
    ops = T()
    N = 64
    x = torch.zeros(1, 8, device="cuda", dtype=torch.float16)
    w = torch.zeros(N, 8, device="cuda", dtype=torch.float16)
    b = torch.linspace(-6, 6, N, device="cuda").half().float().requires_grad_()      # z is the bias, exact in 16 bits
    r = torch.zeros(1, N, device="cuda")
    y = ops.linear_act(x, w, b, r, act)
    (db,) = torch.autograd.grad(y, b, torch.ones_like(y))
    z, step = b.detach().double(), 1e-5
    d = (act_oracle(z + step, act)[0] - act_oracle(z - step, act)[0]) / (2 * step)
    assert (y.detach()[0].double() - act_oracle(z, act)[0]).abs().max() < 4e-6       # 1.5e-7 of erf, times |z| <= 6, and f32
    assert (db.double() - d).abs().max() < 4e-6


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [1, 40, 300])
def test_linear_act_far_values(act, M):
    """z of infinities, a NaN and the largest values: what the definition gives, forward and slope (z is the bias)"""
    ops = T()
    z = torch.tensor([float("inf"), float("-inf"), float("nan"), 3e38, -3e38, 1e25, -1e25, 100.0, -100.0, 0.0, -0.0, 1e-30, -1e-38, 30.0, -30.0, 8.0],
                     device="cuda").repeat(4)
    x = torch.zeros(M, 8, device="cuda", dtype=torch.bfloat16)
    w = torch.zeros(64, 8, device="cuda", dtype=torch.bfloat16)
    b = z.clone().requires_grad_()
    y = ops.linear_act(x, w, b, torch.zeros(M, 64, device="cuda"), act)
    want, slope = act_oracle(z.double(), act)
    kept, got = y.detach()[M // 2].double(), want
    assert torch.equal(kept.isnan(), got.isnan())
    fine = got.isfinite()
    assert torch.equal(kept[~fine & ~got.isnan()], got[~fine & ~got.isnan()])
    assert ((kept - got)[fine].abs() <= 1e-5 * got[fine].abs() + 1e-5).all()      # (1.5e-7 of erf times |z| = 30, and f32)
    (db,) = torch.autograd.grad(y, b, torch.ones_like(y))
    far = {"none": (1.0, 1.0)}.get(act, (1.0, 0.0))      # at the infinities: the limits
    slope = torch.where(z == math.inf, far[0], torch.where(z == -math.inf, far[1], slope))
    assert torch.equal(db.isnan(), z.isnan() & (act != "none"))
    assert ((db.double() / M - slope)[~z.isnan()].abs() < 1e-4).all()


@pytest.mark.gpu
def test_linear_act_options():
    ops, g = T(), gen(21)
    x, w, b, r = linear_case(g, 37, 64, 48, torch.bfloat16, torch.float32, True)
    full = ops.linear_act(x, w, b, r, "silu")
    z = x.double() @ w.double().t() + b.double()
    close(full, act_oracle(z, "silu")[0] + r.double(), 1.2 * (x.double().abs() @ w.double().abs().t() + b.double().abs()) + r.double().abs())
    assert torch.equal(ops.linear_act(x.view(1, 37, 64), w, b, r.view(1, 37, 48), "silu")[0], full)
    wide, wwide = randn(g, 37, 200, dtype=torch.bfloat16), randn(g, 96, 200, dtype=torch.bfloat16)
    for lo in (0, 8, 3):        # strided rows on 16 bytes are used as they are, others are copied
        wide[:, lo:lo + 64], wwide[::2, lo:lo + 64] = x, w
        assert torch.equal(ops.linear_act(wide[:, lo:lo + 64], wwide[::2, lo:lo + 64], b, r, "silu"), full)
    rr = torch.zeros(37, 51, device="cuda")
    rr[:, 2:50] = r
    assert torch.equal(ops.linear_act(x, w, b, rr[:, 2:50], "silu"), full)
    # each gradient alone equals the one among all
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b, r)]
    dy = randn(g, 37, 48)
    want = torch.autograd.grad(ops.linear_act(*leaves, "silu"), leaves, dy)
    for k in range(4):
        one = [t.detach().clone().requires_grad_(j == k) for j, t in enumerate((x, w, b, r))]
        assert torch.equal(torch.autograd.grad(ops.linear_act(*one, "silu"), one[k], dy)[0], want[k])
    assert want[2].dtype == torch.float32
    e = x[:0].clone().requires_grad_()
    wg = w.clone().requires_grad_()
    y = ops.linear_act(e, wg, b, None, "gelu")
    de, dw = torch.autograd.grad(y, (e, wg), torch.zeros_like(y))
    assert y.shape == (0, 48) and de.shape == e.shape and not dw.any()
    # an operand's infinity reaches its row alone, and K's last piece brings in nothing behind it
    x[5, 63] = float("inf")
    y = ops.linear_act(x, w, b)
    assert not y[5].isfinite().any() and y[:5].isfinite().all() and y[6:].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("res", ["none", "half", "f32"])
@pytest.mark.parametrize("M,K,N", [(m, (k + 15) // 16 * 16, n) for m, k, n in LINEAR])
def test_linear_fp8(M, K, N, res):
    ops, g = T(), gen(M + K + N + 1)
    act = ACTS[(M + N + len(res)) % 5]
    dtype = HALF[(M + N) % 2]
    rt = {"none": None, "half": dtype, "f32": torch.float32}[res]
    x, w, b, r = linear_case(g, M, K, N, dtype, rt, bool(M % 2))
    (xq, xs), (wq, ws) = ops.quantize_fp8(x), ops.quantize_fp8(w)
    y = ops.linear_fp8(xq, xs, wq, ws, b, r, act, dtype)
    xd, wd = xq.double() * xs.double()[:, None], wq.double() * ws.double()[:, None]
    z = xd @ wd.t() + b.double()
    zmag = xd.abs() @ wd.abs().t() + b.double().abs()
    rd = torch.zeros_like(z) if r is None else r.double()
    close(y, act_oracle(z, act)[0] + rd, 1.2 * zmag + rd.abs(), "y", F32 if res == "f32" else F8)
    assert y.dtype == (rt or dtype)
    if res == "none":
        close(ops.linear_fp8(xq, xs, wq, ws, None, None, "none", torch.float32), xd @ wd.t(), zmag)


# ------------------------------------------------------------------ together, as a block uses them
def block(ops, x, branch, p, pos, freq, B, N, H, prefix):
    """attention's half of a pre-norm block: the last branch joins the stream, norm, q | k | v, rotary, attention, projection onto the stream"""
    D = x.shape[-1]
    y, h = ops.add_rms_norm(branch, x, p["n"])
    qkv = ops.linear_act(y, p["wqkv"], p["bqkv"])
    qkv = ops.rotary(qkv.view(B, N, 3 * H, D // H), pos, freq, [8, 8], 2 * H, prefix).view(B, N, 3 * D)
    a = ops.attention(qkv, H)
    h = ops.linear_act(a, p["wo"], p["bo"], h)
    u = ops.linear_act(ops.rms_norm(h, p["n2"], out_dtype=torch.bfloat16), p["w1"], p["b1"], None, "gelu")
    return ops.linear_act(u, p["w2"], p["b2"], h)


def block_oracle(x, branch, p, pos, freq, B, N, H, prefix):
    D = x.shape[-1]
    h = x + branch
    y = norm_oracle(h, p["n"], 1e-6)[0]
    qkv = (y @ p["wqkv"].t() + p["bqkv"]).view(B, N, 3 * H, D // H)
    axis = torch.tensor([0] * 8 + [1] * 8, device=x.device)
    ang = pos.double()[:, axis] * freq
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    v = qkv[:, prefix:, :2 * H]
    v = torch.cat((v[..., :16] * c - v[..., 16:] * s, v[..., 16:] * c + v[..., :16] * s), -1)
    qk = torch.cat((qkv[:, :prefix, :2 * H], v), 1)
    q, k = qk[:, :, :H].transpose(1, 2), qk[:, :, H:].transpose(1, 2)
    a = torch.softmax(q @ k.transpose(2, 3) * (D // H) ** -0.5, -1) @ qkv[:, :, 2 * H:].transpose(1, 2)
    h = h + a.transpose(1, 2).reshape(B, N, D) @ p["wo"].t() + p["bo"]
    u = act_oracle(norm_oracle(h, p["n2"], 1e-6)[0] @ p["w1"].t() + p["b1"], "gelu")[0]
    return h + u @ p["w2"].t() + p["b2"]


def block_inputs(B=2, grid=6, prefix=5, D=96, H=3, hid=256):
    g = gen(77)
    N = prefix + grid * grid
    ops = T()
    p = {"n": 1 + 0.1 * randn(g, D), "n2": 1 + 0.1 * randn(g, D)}
    for name, (o, i) in {"qkv": (3 * D, D), "o": (D, D), "1": (hid, D), "2": (D, hid)}.items():
        p["w" + name], p["b" + name] = randn(g, o, i, dtype=torch.bfloat16, scale=i ** -0.5), randn(g, o, dtype=torch.bfloat16, scale=0.1)
    x, branch = randn(g, B, N, D), randn(g, B, N, D, dtype=torch.bfloat16, scale=0.5)
    return x, branch, p, ops.grid_positions(grid, grid, device="cuda"), ops.rotary_frequencies([8, 8], 100.0, device="cuda"), B, N, H, prefix


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.gpu
def test_block_forward_backward_against_64_bits():
    ops = T()
    x, branch, p, *rest = block_inputs()
    leaves = [x, branch, *p.values()]
    for t in leaves:
        t.requires_grad_()
    y = block(ops, x, branch, p, *rest)
    dy = randn(gen(78), *y.shape)
    got = torch.autograd.grad(y, leaves, dy)
    ref = {k: v.detach().double().requires_grad_() for k, v in p.items()}
    xr, br = x.detach().double().requires_grad_(), branch.detach().double().requires_grad_()
    yr = block_oracle(xr, br, ref, *rest)
    want = torch.autograd.grad(yr, [xr, br, *ref.values()], dy.double())
    # nine roundings to bf16 lie on the longest way (2^-9 each in the mean, uncorrelated): 3 * 2^-8 of the branches, of which the stream keeps 1
    assert rel(y.detach(), yr.detach()) < 6e-3
    for name, a, b in zip(["x", "branch", *p], got, want):
        assert rel(a, b) < 2.5e-2, (name, rel(a, b))


@pytest.mark.gpu
def test_serving_block_in_8_bits():
    """norm -> 8 bits -> q | k | v, attention -> 8 bits -> projection onto the stream, against the same steps in 64 bits on the same 8 bits"""
    ops = T()
    x, branch, p, pos, freq, B, N, H, prefix = block_inputs()
    D = x.shape[-1]
    wq, ws = ops.quantize_fp8(p["wqkv"])
    oq, os_ = ops.quantize_fp8(p["wo"])
    q, s, h = ops.add_rms_norm_fp8(branch, x, p["n"])
    qkv = ops.linear_fp8(q, s, wq, ws, p["bqkv"])
    want = (q.double() * s.double()[..., None]) @ (wq.double() * ws.double()[:, None]).t() + p["bqkv"].double()
    assert rel(qkv, want) < 2 ** -8
    ops.rotary_(qkv.view(B, N, 3 * H, D // H), pos, freq, [8, 8], 2 * H, prefix)
    a = ops.attention(qkv, H)
    aq, as_ = ops.quantize_fp8(a)
    y = ops.linear_fp8(aq, as_, oq, os_, p["bo"], h)
    want = h.double() + (aq.double() * as_.double()[..., None]) @ (oq.double() * os_.double()[:, None]).t() + p["bo"].double()
    assert y.dtype == torch.float32 and rel(y, want) < 1e-6
    full = block_oracle(x.double(), branch.double(), {k: v.double() for k, v in p.items()}, pos, freq, B, N, H, prefix)
    assert full.shape == y.shape


# ------------------------------------------------------------------ streams, graphs, modes
@pytest.mark.gpu
def test_other_streams_and_threads():
    import threading
    ops = T()
    args = block_inputs()
    want = block(ops, *args)
    torch.cuda.synchronize()
    got = {}

    def work(k):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s), torch.no_grad():
            for _ in range(5):
                got[k] = block(ops, *args)
        s.synchronize()
    threads = [threading.Thread(target=work, args=(k,)) for k in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(v, want) for v in got.values()) and len(got) == 3


@pytest.mark.gpu
def test_captured_and_replayed():
    """serving steps and a training step in graphs, two of them alive at once, replayed between eager work: each replay as the eager result"""
    ops = T()
    x, branch, p, pos, freq, B, N, H, prefix = block_inputs()
    wq, ws = ops.quantize_fp8(p["wqkv"])
    w = p["n"].clone().requires_grad_()
    w1, b1 = p["w1"].clone().requires_grad_(), p["b1"].clone().requires_grad_()
    dy = randn(gen(5), B, N, p["w1"].shape[0], dtype=torch.bfloat16)

    def serve():
        q, s, h = ops.add_rms_norm_fp8(branch, x, p["n"])
        qkv = ops.linear_fp8(q, s, wq, ws, p["bqkv"])
        return ops.rotary(qkv.view(B, N, 3 * H, -1), pos, freq, [8, 8], 2 * H, prefix), h

    def train():
        y, h = ops.add_rms_norm(branch, x, w)
        u = ops.linear_act(y, w1, b1, None, "silu")
        return (u.detach(), *torch.autograd.grad(u, (w, w1, b1), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for f in (serve, train, serve, train):
            f()
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = f()
            graphs.append((g, f, out))
    torch.cuda.current_stream().wait_stream(side)
    for turn in range(4):
        x.copy_(randn(gen(100 + turn), *x.shape))
        branch.copy_(randn(gen(200 + turn), *x.shape, dtype=branch.dtype))
        for g, f, out in graphs:
            g.replay()
        for g, f, out in graphs:
            want = f()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
def test_inside_another_operand_mode():
    """the tensors' type decides which library runs, whatever mode the thread is in"""
    from miphei_vit_amd import _lib
    ops, g = T(), gen(31)
    for dtype in HALF:
        x, w = randn(g, 20, 64, dtype=dtype), randn(g, 40, 64, dtype=dtype)
        want = (ops.linear_act(x, w), ops.rms_norm(x, torch.ones(64, device="cuda")), *ops.quantize_fp8(x))
        for mode in ("bf16", "f16"):
            with _lib.operands(mode):
                got = (ops.linear_act(x, w), ops.rms_norm(x, torch.ones(64, device="cuda")), *ops.quantize_fp8(x))
                assert _lib.operand_mode() == mode
            assert all(torch.equal(a.float(), b.float()) for a, b in zip(got, want))


@pytest.mark.gpu
def test_gradient_of_a_gradient_is_refused():
    ops, g = T(), gen(41)
    x, w = randn(g, 4, 64).requires_grad_(), randn(g, 64).requires_grad_()
    (dx,) = torch.autograd.grad(ops.rms_norm(x, w).sum(), x, create_graph=False)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(ops.rms_norm(x, w).square().sum(), x, create_graph=True)
    a, b = randn(g, 4, 64, dtype=torch.float16).requires_grad_(), randn(g, 32, 64, dtype=torch.float16).requires_grad_()
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(ops.linear_act(a, b).square().sum(), a, create_graph=True)


@pytest.mark.gpu
def test_traced_by_the_compiler_front_end():
    """one graph without breaks through the shape implementations, with the eager results"""
    ops, g = T(), gen(42)
    x, r, w = randn(g, 6, 64, dtype=torch.bfloat16), randn(g, 6, 64), randn(g, 64)
    wt, b = randn(g, 96, 64, dtype=torch.bfloat16), randn(g, 96, dtype=torch.bfloat16)
    pos, freq = torch.arange(6, device="cuda", dtype=torch.int32)[:, None], ops.rotary_frequencies([16], device="cuda")

    def f(x, r, w, wt, b):
        y, h = ops.add_rms_norm(x, r, w)
        z = ops.linear_act(y, wt, b, None, "silu").view(1, 6, 3, 32)
        return ops.rotary(z, pos, freq, [16], 2), h, *ops.quantize_fp8(y.detach())
    want = f(x, r, w, wt, b)
    got = torch.compile(f, backend="aot_eager", fullgraph=True)(x, r, w, wt, b)
    assert all(torch.equal(u.float(), v.float()) for u, v in zip(want, got))


@pytest.mark.gpu
def test_saved_tensors_changed_in_place_are_noticed():
    ops, g = T(), gen(43)
    x, r, w = randn(g, 4, 64).requires_grad_(), randn(g, 4, 64), randn(g, 64).requires_grad_()
    y, h = ops.add_rms_norm(x, r, w)
    h.detach().add_(1)                                      # (the stream that the backward pass reads)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    q = randn(g, 1, 3, 2, 8, dtype=torch.float16)
    p = (q.clone().requires_grad_() * 1)
    z = p * p
    with torch.no_grad():
        ops.rotary_(p, torch.zeros(3, 1, device="cuda", dtype=torch.int32), torch.ones(4, device="cuda"), [4])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()


# ------------------------------------------------------------------ calls that the documentation allows, at its edges
def test_shapes_of_sizes_that_vary():
    """the shape implementations with a symbolic number of rows, as a compiled model is traced for other batch sizes"""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.symbolic_shapes import DimDynamic, ShapeEnv, StatelessSymbolicContext
    ops, mode = T(), FakeTensorMode(shape_env=ShapeEnv())
    x = mode.from_tensor(torch.empty(6, 64, dtype=torch.bfloat16, device="meta"),
                         symbolic_context=StatelessSymbolicContext(dynamic_sizes=[DimDynamic.DYNAMIC, DimDynamic.STATIC]))
    rows = x.shape[0]
    assert not isinstance(rows, int)
    with mode:
        w, lw, b = (torch.empty(*s, device="meta") for s in ((64,), (48, 64), (48,)))
        y, h = ops.add_rms_norm(x, x.float(), w)
        assert y.shape == (rows, 64) and h.shape == (rows, 64) and y.shape[0] is not int
        (q, s), (wq, ws) = ops.quantize_fp8(y), ops.quantize_fp8(lw)
        assert q.shape == (rows, 64) and s.shape == (rows,)
        assert ops.linear_act(x, lw.to(x.dtype), b, None, "gelu").shape == (rows, 48)
        assert ops.linear_fp8(q, s, wq, ws, b, None, "silu").shape == (rows, 48)
        pos, freq = torch.empty(x.shape[0], 1, dtype=torch.int32, device="meta"), torch.empty(8, device="meta")
        assert ops.rotary(x.view(1, -1, 4, 16), pos, freq, [8]).shape == (1, rows, 4, 16)
        with pytest.raises(ValueError, match="mvit::"):
            ops.linear_act(x, lw[:, :56].to(x.dtype))


def test_rotary_of_overlapping_windows():
    """heads that are sliding windows of one row: an input may overlap, what is written may not"""
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops = T()
    with FakeTensorMode():
        x = fake(2, 7, 20).unfold(2, 16, 1)
        p, fr = fake(7, 1, dtype=torch.int32), fake(8, dtype=torch.float32)
        assert x.stride()[2:] == (1, 1)
        y = ops.rotary(x, p, fr, [8])
        assert y.shape == x.shape and y.stride(3) == 1 and y.is_contiguous()
        for z in (x, fake(2, 7, 36).unfold(2, 16, 4), fake(2, 5, 3, 16).expand(2, 5, 3, 16)[:, :1].expand(2, 7, 3, 16)):
            with pytest.raises(ValueError, match="in place"):
                ops.rotary_(z, p, fr, [8])
        ops.rotary_(fake(7, 2, 3, 16).transpose(0, 1), p, fr, [8])      # apart in any order
        ops.rotary_(fake(2, 7, 5, 32)[:, :, ::2, 8:24], p, fr, [8])


@pytest.mark.gpu
def test_rotary_of_overlapping_windows_on_the_gpu():
    ops, g = T(), gen(51)
    x = randn(g, 2, 7, 20, dtype=torch.bfloat16).unfold(2, 16, 1)
    p, fr = torch.arange(7, device="cuda", dtype=torch.int32)[:, None], ops.rotary_frequencies([8], device="cuda")
    for il in (False, True):
        assert torch.equal(ops.rotary(x, p, fr, [8], interleaved=il), ops.rotary(x.contiguous(), p, fr, [8], interleaved=il))


@pytest.mark.gpu
def test_positions_and_frequencies_have_no_gradient():
    ops = T()
    x = torch.randn(1, 3, 2, 8, device="cuda")
    p, fr = torch.zeros(3, 1, device="cuda"), torch.ones(4, device="cuda")
    for a, b in ((p.clone().requires_grad_(), fr), (p, fr.clone().requires_grad_())):
        for f in (ops.rotary, ops.rotary_):
            with pytest.raises(RuntimeError, match="no gradient"):
                f(x, a, b, [4])
        with torch.no_grad():
            ops.rotary(x, a, b, [4])


@pytest.mark.gpu
def test_backward_operators_refuse_what_does_not_belong_together():
    m = torch.ops.mvit
    x, w, dy = (torch.zeros(*s, device="cuda", dtype=torch.bfloat16) for s in ((4, 16), (8, 16), (4, 8)))
    for args in ((dy[:3], x, w, dy, "gelu"), (dy, x, w, dy[:3], "gelu"), (dy, x, w, x.new_empty(0), "silu"), (dy, x, w, dy.float(), "silu"),
                 (dy, x, w[:, :8], dy, "none"), (dy, x.half(), w, dy, "none")):
        with pytest.raises(ValueError, match="mvit::"):
            m.linear_act_backward(*args, True, True, True, torch.float32)
    v, rstd = torch.ones(16, device="cuda"), torch.ones(4, device="cuda")
    for args in ((x[:3], None, x, v, rstd), (x, x[:3], x, v, rstd), (x, None, x, v[:8], rstd), (x, None, x, v, rstd[:3]), (x, None, x, v, rstd.cpu())):
        with pytest.raises(ValueError, match="mvit::"):
            m.rms_norm_backward(*args, torch.bfloat16, True, False, True)


@pytest.mark.gpu
def test_compiled_at_several_batch_sizes():
    """one compiled model, forward and backward, at batch sizes that it was not traced with; the in-place turn among its operators"""
    ops, g = T(), gen(52)
    w, wt, b = randn(g, 64), randn(g, 96, 64, dtype=torch.bfloat16), randn(g, 96)
    freq = ops.rotary_frequencies([16], device="cuda")

    def f(x, r, w, wt, b, pos):
        y, h = ops.add_rms_norm(x, r, w)
        z = ops.linear_act(y, wt, b, None, "gelu")
        return ops.rotary(z.view(1, -1, 3, 32), pos, freq, [16], 2), h

    def serve(x, wt, pos):
        q, s = ops.quantize_fp8(x)
        z = ops.linear_fp8(q, s, *ops.quantize_fp8(wt)).view(1, -1, 3, 32)
        return ops.rotary_(z, pos, freq, [16], 2) * 2
    cf = torch.compile(f, backend="aot_eager", fullgraph=True, dynamic=True)
    cs = torch.compile(serve, backend="aot_eager", fullgraph=True, dynamic=True)
    for M in (6, 9, 40):
        x, r = randn(g, M, 64, dtype=torch.bfloat16), randn(g, M, 64)
        pos = torch.arange(M, device="cuda", dtype=torch.int32)[:, None]
        leaves = [t.clone().requires_grad_() for t in (x, r, w, wt, b)]
        results = []
        for fn in (f, cf):
            y, h = fn(*leaves, pos)
            results.append((y.detach(), h.detach(), *torch.autograd.grad((y.float().square().sum() + h.sum()), leaves)))
        assert all(torch.equal(u, v) for u, v in zip(*results))
        assert torch.equal(serve(x, wt, pos), cs(x, wt, pos))


@pytest.mark.gpu
def test_operators_keep_their_schemas():
    """what torch itself checks of an operator: nothing written that is not declared, shapes as traced, autograd where it belongs"""
    g, m = gen(53), torch.ops.mvit
    x, r, w = randn(g, 6, 64, dtype=torch.bfloat16), randn(g, 6, 64), randn(g, 64)
    wt, b = randn(g, 96, 64, dtype=torch.bfloat16), randn(g, 96)
    z, pos, freq = randn(g, 1, 6, 3, 32), torch.arange(6, device="cuda")[:, None], torch.rand(16, device="cuda")
    q, s = m.quantize_fp8(x)
    wq, ws = m.quantize_fp8(wt)
    grad = lambda *ts: [t.clone().requires_grad_() for t in ts]  # noqa: E731
    for name, args in (("rms_norm_forward", (*grad(x, r, w), 1e-6, None)), ("rms_norm_forward", (x, None, w, 1e-6, None)),
                       ("rms_norm_fp8", (x, r, w, 1e-6)), ("quantize_fp8", (x,)), ("rotary_forward", (*grad(z), pos, freq, [16], 2, 1 - 1, False, False)),
                       ("rotary_", (z, pos, freq, [16], 2, 0, False)), ("linear_act_forward", (*grad(x, wt, b, r.repeat(1, 2)[:, :96]), "silu", False)),
                       ("linear_fp8", (q, s, wq, ws, b, None, "gelu", torch.bfloat16))):
        # (torch's schema check compares by arithmetic that it does not have for e4m3 tensors)
        utils = ("test_autograd_registration", "test_faketensor") + (() if "fp8" in name else ("test_schema",))
        torch.library.opcheck(getattr(m, name).default, args, test_utils=utils)


@pytest.mark.gpu
def test_linear_fp8_operands_in_place():
    """8-bit operands as slices: on 16 bytes as they are, else copied; scales with strides"""
    ops, g = T(), gen(54)
    for M in (3, 45):
        (q, s), (wq, ws) = ops.quantize_fp8(randn(g, M, 64)), ops.quantize_fp8(randn(g, 40, 64))
        want = ops.linear_fp8(q, s, wq, ws)
        for lo in (0, 16, 5):
            wide, wwide = torch.zeros(M, 2, 96, device="cuda").to(q.dtype), torch.zeros(80, 96, device="cuda").to(q.dtype)
            wide.view(torch.uint8)[:, 1, lo:lo + 64] = q.view(torch.uint8)
            wwide.view(torch.uint8)[::2, lo:lo + 64] = wq.view(torch.uint8)
            ss = torch.stack((s, s), 1)[:, 1]
            assert torch.equal(ops.linear_fp8(wide[:, 1, lo:lo + 64], ss, wwide[::2, lo:lo + 64], ws.repeat_interleave(2)[::2]), want)


@pytest.mark.gpu
def test_rows_far_apart():
    """row strides up to 2^23 bytes, the most that is used without a copy: offsets of a tile's 256 rows up to 31 bits"""
    ops, g = T(), gen(55)
    M, N = 1030, 4608
    for es, stride in ((2, 2 ** 22), (1, 2 ** 23)):
        big = torch.empty(M, stride, device="cuda", dtype=torch.bfloat16 if es == 2 else torch.float8_e4m3fn)
        x, w = randn(g, M, 64, dtype=torch.bfloat16), randn(g, N, 64, dtype=torch.bfloat16)
        if es == 2:
            big[:, -64:] = x
            assert torch.equal(ops.linear_act(big[:, -64:], w), ops.linear_act(x, w))
            dy, w = randn(g, M, N, dtype=torch.bfloat16), w.requires_grad_()
            assert torch.equal(torch.autograd.grad(ops.linear_act(big[:, -64:], w), w, dy)[0], torch.autograd.grad(ops.linear_act(x, w), w, dy)[0])
            w = w.detach()
        else:
            (q, s), (wq, ws) = ops.quantize_fp8(x), ops.quantize_fp8(w)
            big.view(torch.uint8)[:, -64:] = q.view(torch.uint8)
            for out in (torch.bfloat16, torch.float32):
                assert torch.equal(ops.linear_fp8(big[:, -64:], s, wq, ws, out_dtype=out), ops.linear_fp8(q, s, wq, ws, out_dtype=out))
        del big


@pytest.mark.gpu
def test_long_offsets():
    """more than 2^31 elements: the last rows as a small call gives them, forward and backward"""
    ops, g = T(), gen(56)
    M, D = 2 ** 17 + 5, 16384
    tail = slice(M - 8, M)
    x = torch.zeros(M, D, device="cuda", dtype=torch.bfloat16)
    x[tail] = randn(g, 8, D, dtype=torch.bfloat16)
    w = randn(g, D)
    few = x[tail].clone().requires_grad_()
    q, s = ops.quantize_fp8(x)
    q8, s8 = ops.quantize_fp8(few.detach())
    assert torch.equal(q[tail].view(torch.uint8), q8.view(torch.uint8)) and torch.equal(s[tail], s8) and not q[:8].view(torch.uint8).any()
    del q, s
    dy = torch.zeros_like(x)
    dy[tail] = randn(g, 8, D, dtype=torch.bfloat16)
    x.requires_grad_()
    y = ops.rms_norm(x, w)
    y8 = ops.rms_norm(few, w)
    (dx,), (dx8,) = torch.autograd.grad(y, x, dy), torch.autograd.grad(y8, few, dy[tail])
    assert torch.equal(y.detach()[tail], y8.detach()) and torch.equal(dx[tail], dx8) and not dx[:8].any()
    del x, y, dx, dy
    M, K, N = 2 ** 17 + 5, 16, 16400
    tail = slice(M - 5, M)
    x, w, b = randn(g, M, K, dtype=torch.bfloat16), randn(g, N, K, dtype=torch.bfloat16).requires_grad_(), randn(g, N).requires_grad_()
    r = torch.ones(M, N, device="cuda", dtype=torch.bfloat16)
    x.requires_grad_()
    y = ops.linear_act(x, w, b, r, "silu")
    dy = torch.zeros_like(r)
    dy[tail] = randn(g, 5, N, dtype=torch.bfloat16)
    got = torch.autograd.grad(y, (x, w, b), dy)
    few = x.detach()[tail].clone().requires_grad_()
    y5 = ops.linear_act(few, w, b, r[tail], "silu")
    want = torch.autograd.grad(y5, (few, w, b), dy[tail])
    for u, v in zip((y.detach()[tail], got[0][tail], *got[1:]), (y5.detach(), *want)):
        # other kernels, other orders of the same sums: the kept z may round to the neighbouring 16-bit value, which moves dz by at most a unit
        # of z times silu'' <= 2^-7 * 0.31 times |dy| <= 5, times |x| or |w| <= 5: 0.06; and a unit of the result's own rounding
        assert ((u.float() - v.float()).abs() <= 2.0 ** -7 * v.float().abs() + 0.06).all()
    assert not got[0][:8].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("M,K,N", [(20816, 512, 64), (20815, 64, 60), (33, 1536, 4096), (1, 1536, 4096), (5264, 1536, 1536), (700, 512, 4100), (200, 72, 2568)])
def test_linear_act_gradients_of_few_tiles(M, K, N, dtype):
    """products whose K axis is taken in parts: all rows of a small weight, all columns of few rows; the same every time"""
    ops, g = T(), gen(M + K + N)
    x, w = randn(g, M, K, dtype=dtype).requires_grad_(), randn(g, N, K, dtype=dtype, scale=K ** -0.5).requires_grad_()
    dy = randn(g, M, N, dtype=dtype)
    y = ops.linear_act(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    d, xd, wd = dy.double(), x.detach().double(), w.detach().double()
    close(dx, d @ wd, d.abs() @ wd.abs(), "dx")
    close(dw, d.t() @ xd, d.abs().t() @ xd.abs(), "dw")
    again = torch.autograd.grad(y, (x, w), dy)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "gelu"])
@pytest.mark.parametrize("N", [72, 75])
def test_linear_act_gradients_of_odd_upstream_layouts(N, act):
    """a gradient that is one value off 16 bytes, transposed, expanded or f32 gives what its dense copy gives"""
    ops, g = T(), gen(57 + N)
    M, K = 70, 40
    x, w, b = randn(g, M, K, dtype=torch.bfloat16).requires_grad_(), randn(g, N, K, dtype=torch.bfloat16).requires_grad_(), randn(g, N).requires_grad_()
    y = ops.linear_act(x, w, b, None, act)
    dy = randn(g, M, N, dtype=torch.bfloat16)
    want = torch.autograd.grad(y, (x, w, b), dy, retain_graph=True)
    off = torch.zeros(M * N + 1, device="cuda", dtype=torch.bfloat16)[1:].view(M, N).copy_(dy)
    for d in (off, dy.t().contiguous().t()):
        for u, v in zip(torch.autograd.grad(y, (x, w, b), d, retain_graph=True), want):
            # (db's sums go in another order where the gradient is taken by elements: 70 values of at most 5 each)
            assert torch.equal(u, v) if u.dtype == torch.bfloat16 else ((u - v).abs() <= 70 * 5 * 70 * 2.0 ** -24).all()
    row = dy[:1].expand(M, N)
    for u, v in zip(torch.autograd.grad(y, (x, w, b), row, retain_graph=True), torch.autograd.grad(y, (x, w, b), row.contiguous())):
        assert torch.equal(u, v)


LONG_K = [(1, 16384, 512), (1, 16384, 509), (16, 32768, 70), (17, 32768, 136), (30, 16384, 45), (37, 2560, 2044), (64, 7792, 2558), (100, 8192, 64), (33, 4096, 33)]


@pytest.mark.gpu
@pytest.mark.parametrize("res", ["none", "half", "f32"])
@pytest.mark.parametrize("M,K,N", LONG_K)
def test_linear_of_a_long_k(M, K, N, res):
    """few rows and a long K, taken in parts: with a bias, every activation, residuals with strides, the kept pre-activation; twice the same"""
    ops, g = T(), gen(M + K + N)
    dtype = HALF[(M + N) % 2]
    act = ACTS[(M + len(res)) % 5]
    rt = {"none": None, "half": dtype, "f32": torch.float32}[res]
    x, w, b, r = linear_case(g, M, K, N, dtype, rt, bool(N % 2))
    if r is not None:
        wide = torch.zeros(M, N + 3, device="cuda", dtype=rt)
        wide[:, 1:N + 1] = r
        r = wide[:, 1:N + 1]
    z = x.double() @ w.double().t() + b.double()
    mag = x.double().abs() @ w.double().abs().t() + b.double().abs()
    rd = torch.zeros_like(z) if r is None else r.double()
    y = ops.linear_act(x, w, b, r, act)
    close(y, act_oracle(z, act)[0] + rd, 1.2 * mag + rd.abs(), "y")
    assert torch.equal(y, ops.linear_act(x, w, b, r, act))
    out, pre = torch.ops.mvit.linear_act_forward(x, w, b, r, act, True)
    close(pre, z, mag, "pre")
    assert torch.equal(out, y)
    xs, ws = (t.float().abs().amax(-1) / 448 for t in (x, w))          # (rows longer than quantize_fp8 takes)
    xq, wq = ((t.float() / s[:, None]).to(torch.float8_e4m3fn) for t, s in ((x, xs), (w, ws)))
    xd, wd = xq.double() * xs.double()[:, None], wq.double() * ws.double()[:, None]
    z, mag = xd @ wd.t() + b.double(), xd.abs() @ wd.abs().t() + b.double().abs()
    close(ops.linear_fp8(xq, xs, wq, ws, b, r, act, dtype), act_oracle(z, act)[0] + rd, 1.2 * mag + rd.abs(), "fp8", F32 if res == "f32" else F8)


def test_room_for_parts():
    from miphei_vit_amd import _lib
    lib = _lib.lib()
    assert lib.mvit_linear_scratch_bytes(1, 512, 32768) > 0 == lib.mvit_linear_scratch_bytes(1, 1536, 2 * 1536) == lib.mvit_linear_scratch_bytes(5264, 4096, 2 * 1536)
    assert lib.mvit_linear_scratch_bytes(0, 512, 32768) == lib.mvit_linear_scratch_bytes(1, 512, 1 << 24) == 0


# ------------------------------------------------------------------ derivatives of other kinds
def derivative_calls(device):
    """name -> (function of one tensor, that tensor); shapes only where the device is meta"""
    ops, f32, f8 = T(), torch.float32, torch.float8_e4m3fn
    make = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=device)  # noqa: E731
    w, p, fr = make(64, dtype=f32), make(4, 1, dtype=torch.int32), make(8, dtype=f32)
    x, lw, q, wq = make(4, 64), make(32, 64), make(4, 64, dtype=f8), make(32, 64, dtype=f8)
    s, ws = make(4, dtype=f32), make(32, dtype=f32)
    return {
        "rms_norm": (lambda x: ops.rms_norm(x, w), x), "rms_norm weight": (lambda w: ops.rms_norm(x, w), w),
        "add_rms_norm residual": (lambda r: ops.add_rms_norm(x, r, w)[1], x), "linear_act": (lambda x: ops.linear_act(x, lw), x),
        "linear_act weight": (lambda lw: ops.linear_act(x, lw), lw), "linear_act bias": (lambda b: ops.linear_act(x, lw, b), ws),
        "linear_act residual": (lambda r: ops.linear_act(x, lw, None, r), make(4, 32)), "rotary": (lambda x: ops.rotary(x, p, fr, [8]), make(1, 4, 2, 16)),
        "rotary frequencies": (lambda fr: ops.rotary(make(1, 4, 2, 16), p, fr, [8]), fr),
        "rotary_": (lambda x: ops.rotary_(x, p, fr, [8]), make(1, 4, 2, 16)), "quantize_fp8": (lambda x: ops.quantize_fp8(x)[1], x),
        "rms_norm_fp8": (lambda x: ops.rms_norm_fp8(x, w)[1], x), "add_rms_norm_fp8": (lambda x: ops.add_rms_norm_fp8(x, x, w)[2], x),
        "linear_fp8 scale": (lambda s: ops.linear_fp8(q, s, wq, ws), s), "linear_fp8 bias": (lambda b: ops.linear_fp8(q, s, wq, ws, b), ws),
        "linear_fp8 residual": (lambda r: ops.linear_fp8(q, s, wq, ws, None, r), make(4, 32)),
    }


DERIVATIVES = ["rms_norm", "rms_norm weight", "add_rms_norm residual", "linear_act", "linear_act weight", "linear_act bias", "linear_act residual",
               "rotary", "rotary frequencies", "rotary_", "quantize_fp8", "rms_norm_fp8", "add_rms_norm_fp8", "linear_fp8 scale", "linear_fp8 bias",
               "linear_fp8 residual"]


def refuses_other_derivatives(f, x):
    from torch.autograd import forward_ad
    for grad in (True, False):                      # (torch.no_grad() is about the backward pass)
        with forward_ad.dual_level(), torch.set_grad_enabled(grad):
            with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
                f(forward_ad.make_dual(x, torch.ones_like(x)))
    with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
        torch.func.jvp(f, (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError, match="no gradient|functorch"):
        torch.func.grad(lambda x: f(x).float().sum())(x)
    f(x.clone())


@pytest.mark.parametrize("name", DERIVATIVES)
def test_derivatives_that_there_are_not_are_refused(name):
    """forward mode and functional transforms: refused, never a tangent or gradient of zeros"""
    refuses_other_derivatives(*derivative_calls("meta")[name])


@pytest.mark.gpu
@pytest.mark.parametrize("name", DERIVATIVES)
def test_derivatives_that_there_are_not_are_refused_on_the_gpu(name):
    refuses_other_derivatives(*derivative_calls("cuda")[name])


def test_8_bit_operands_that_require_a_gradient_are_refused():
    ops, f32, f8 = T(), torch.float32, torch.float8_e4m3fn
    q, wq, s, ws = (torch.empty(*n, dtype=t, device="meta") for n, t in (((4, 64), f8), ((32, 64), f8), ((4,), f32), ((32,), f32)))
    for a, b in ((q.detach().requires_grad_(), wq), (q, wq.detach().requires_grad_())):
        with pytest.raises(RuntimeError, match="no gradient"):
            ops.linear_fp8(a, s, b, ws)
        with torch.no_grad():
            ops.linear_fp8(a, s, b, ws)


@pytest.mark.gpu
def test_mapped_over_a_batch():
    """torch.vmap of the operators without gradients: each entry as its own call gives it"""
    ops, g = T(), gen(61)
    x, w, lw = randn(g, 3, 4, 64, dtype=torch.bfloat16), randn(g, 64), randn(g, 32, 64, dtype=torch.bfloat16)
    for f in (lambda x: ops.rms_norm(x, w), lambda x: ops.linear_act(x, lw, None, None, "silu"), lambda x: ops.quantize_fp8(x)[1]):
        assert torch.equal(torch.vmap(f)(x), torch.stack([f(v) for v in x]))


# ------------------------------------------------------------------ K in parts of large tiles
# 64 x 64 tiles that leave no room for parts, 128 x 128 tiles that do; ragged ones, and the first row behind the border
LARGE_PARTS = [(513, 14336, 4096), (1400, 8192, 1536), (1297, 8200, 1607)]


@pytest.mark.parametrize("M,K,N", LARGE_PARTS + [(2048, 8192, 1152), (1025, 16384, 2048)])
def test_room_for_parts_of_large_tiles(M, K, N):
    from miphei_vit_amd import _lib
    lib = _lib.lib()
    assert lib.mvit_linear_scratch_bytes(M, N, 2 * K) == 3 * M * N * 4      # 132 to 165 tiles for 256 CUs: three parts make two blocks a CU of most of them
    assert lib.mvit_linear_scratch_bytes(5264, 4096, 2 * 1536) == lib.mvit_linear_scratch_bytes(1301, 1536, 2 * 4096) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("res", ["none", "half", "f32"])
@pytest.mark.parametrize("M,K,N", LARGE_PARTS)
def test_linear_of_a_long_k_in_large_tiles(M, K, N, res):
    """16-bit operands of any K that they take; e4m3 operands of the next multiple of 16"""
    ops, g = T(), gen(M + K + N)
    dtype, act = HALF[(M + N) % 2], ACTS[(M + len(res)) % 5]
    rt = {"none": None, "half": dtype, "f32": torch.float32}[res]
    x, w, b, r = linear_case(g, M, K, N, dtype, rt, bool(N % 2))
    rd = 0 if r is None else r.double()

    def check(y, xd, wd, f32=F32):
        z, mag = xd @ wd.t() + b.double(), xd.abs() @ wd.abs().t() + b.double().abs()
        close(y, act_oracle(z, act)[0] + rd, 1.2 * mag + (0 if r is None else rd.abs()), "y", f32)
    y = ops.linear_act(x, w, b, r, act)
    check(y, x.double(), w.double())
    assert torch.equal(y, ops.linear_act(x, w, b, r, act))
    x, w = (torch.nn.functional.pad(t, (0, -K % 16)) for t in (x, w))
    xs, ws = (t.float().abs().amax(-1) / 448 for t in (x, w))          # (rows longer than quantize_fp8 takes)
    xq, wq = ((t.float() / s[:, None]).to(torch.float8_e4m3fn) for t, s in ((x, xs), (w, ws)))
    check(ops.linear_fp8(xq, xs, wq, ws, b, r, act, dtype), xq.double() * xs.double()[:, None], wq.double() * ws.double()[:, None], F32 if res == "f32" else F8)


# ------------------------------------------------------------------ the value in front of the activation
def pre_of_all_modes(device):
    g = torch.Generator(device=device).manual_seed(62) if device == "cuda" else None
    make = (lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()) if g else (lambda *s: torch.empty(*s, device=device, dtype=torch.bfloat16))  # noqa: E731
    for act in ("none", "gelu"):
        for wants in ((), (0,), (1,), (2,), (3,), (0, 1, 2, 3)):
            args = [t.requires_grad_(k in wants) for k, t in enumerate((make(5, 64), make(24, 64), make(24), make(5, 24)))]
            yield act, wants, args, torch.ops.mvit.linear_act_forward(*args, act, True)


def test_pre_activation_is_given_where_it_is_asked_for():
    for act, wants, _, (y, pre) in pre_of_all_modes("meta"):
        assert pre.shape == y.shape == (5, 24), (act, wants)
        assert y.requires_grad == bool(wants) and not pre.requires_grad


@pytest.mark.gpu
def test_pre_activation_is_given_where_it_is_asked_for_on_the_gpu():
    for act, wants, (x, w, b, r), (y, pre) in pre_of_all_modes("cuda"):
        x, w, b = (t.detach().double() for t in (x, w, b))
        close(pre, x @ w.t() + b, x.abs() @ w.abs().t() + b.abs(), f"{act} {wants}")
        if wants:
            y.backward(torch.ones_like(y))


# ------------------------------------------------------------------ the norm's backward pass: widths between the layouts' borders, types
@pytest.mark.gpu
@pytest.mark.parametrize("types", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16)], ids=str)
@pytest.mark.parametrize("M,D", [(2047, 520), (2049, 520), (4100, 768), (4095, 1053), (2050, 1280), (2050, 1281), (8200, 1100)])
def test_rms_norm_between_the_layouts(M, D, types):
    test_rms_norm_forward_backward(M, D, types)


@pytest.mark.gpu
@pytest.mark.parametrize("res", [False, True])
@pytest.mark.parametrize("out", HALF)
@pytest.mark.parametrize("M,D", [(1, 1), (5, 512), (1037, 520), (70, 1531), (40, 4096), (9, 8192), (2, 16383), (4097, 64)])
def test_rms_norm_of_an_f32_stream_with_a_16_bit_output(M, D, out, res):
    """the second norm of a block: dy in 16 bits, everything else in f32"""
    ops, g = T(), gen(M * 13 + D)
    x, w = randn(g, M, D).requires_grad_(), (1 + 0.2 * randn(g, D)).requires_grad_()
    dy = randn(g, M, D, dtype=out)
    if res:
        r, dh = randn(g, M, D, scale=3).requires_grad_(), randn(g, M, D)
        y, h = ops.add_rms_norm(x, r, w, 1e-5, out_dtype=out)
        close(h.detach(), x.detach().double() + r.detach().double(), x.detach().double().abs() + r.detach().double().abs(), "h")
        dx, dr, dw = torch.autograd.grad((y, h), (x, r, w), (dy, dh))
        assert torch.equal(dx, dr)
    else:
        y, h, dh = ops.rms_norm(x, w, 1e-5, out_dtype=out), x, None
        dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert y.dtype == out and dx.dtype == dw.dtype == torch.float32
    hd, wd, dyd = h.detach().double(), w.detach().double(), dy.double()
    want, rstd = norm_oracle(hd, wd, 1e-5)
    close(y.detach(), want, want.abs(), "y")
    xhat, wdy = hd * rstd, wd * dyd
    base = 0 if dh is None else dh.double()
    close(dx, base + rstd * (wdy - xhat * (wdy * xhat).mean(-1, keepdim=True)),
          (0 if dh is None else dh.double().abs()) + rstd * (wdy.abs() + xhat.abs() * (wdy * xhat).abs().mean(-1, keepdim=True)), "dx")
    close(dw, (dyd * xhat).sum(0), (dyd * xhat).abs().sum(0), "dweight")


# ------------------------------------------------------------------ what stood in the tests above without being asked
@pytest.mark.parametrize("sections", [[], [0], [0, 0]], ids=str)
def test_rotary_without_sections_is_refused(sections):
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops = T()
    with FakeTensorMode():
        x, n = fake(2, 7, 6, 16), len(sections)
        for f in (ops.rotary, ops.rotary_):
            with pytest.raises(ValueError, match="sections"):
                f(x, fake(7, n, dtype=torch.int32), fake(0, dtype=torch.float32), sections)


def test_a_varying_number_of_rows_stays_one():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.symbolic_shapes import DimDynamic, ShapeEnv, StatelessSymbolicContext
    ops, mode = T(), FakeTensorMode(shape_env=ShapeEnv())
    x = mode.from_tensor(torch.empty(6, 64, dtype=torch.bfloat16, device="meta"),
                         symbolic_context=StatelessSymbolicContext(dynamic_sizes=[DimDynamic.DYNAMIC, DimDynamic.STATIC]))
    with mode:
        y, h = ops.add_rms_norm(x, x.float(), torch.empty(64, device="meta"))
        q, s = ops.quantize_fp8(y)
        z = ops.linear_act(x, torch.empty(48, 64, device="meta", dtype=torch.bfloat16))
    for t in (y, h, q, s, z):
        assert isinstance(t.shape[0], torch.SymInt), t.shape      # (a plain int here would be a size that the trace has fixed)


@pytest.mark.gpu
def test_serving_block_in_8_bits_against_64_bits():
    """attention's half of a block in 8 bits, each step against 64 bits on what it was given, and all of it against the unquantised block.

    The whole: e4m3 with a scale a row is off by at most 2^-4 of a value above its normal range, uniformly spread in its step: on the average of
    values 2^-4 / sqrt 3 relative at the bottom of a binade, half of that at its top, 0.027 of a tensor's norm (2^-4 / sqrt 3 * 0.75).  A product of
    two such operands, of random signs, is off by 0.027 sqrt 2 = 0.038 of its norm.  q, k and v carry it; the softmax averages v over 41 keys, their
    errors with it, and turns the scores' error, 0.038 sqrt 2 of scores of unit size, into as much of its weights, uncorrelated with v: 0.038 + 0.054 in
    quadrature 0.066.  The projection quantises twice more (0.038): 0.076 of the branch's norm.  Three times that bounds it."""
    ops = T()
    x, branch, p, pos, freq, B, N, H, prefix = block_inputs()
    D = x.shape[-1]
    Dh = D // H
    wq, ws = ops.quantize_fp8(p["wqkv"])
    oq, os_ = ops.quantize_fp8(p["wo"])
    with torch.no_grad():
        q, s, h = ops.add_rms_norm_fp8(branch, x, p["n"])
        qkv = ops.linear_fp8(q, s, wq, ws, p["bqkv"])
        before = qkv.clone()
        ops.rotary_(qkv.view(B, N, 3 * H, Dh), pos, freq, [8, 8], 2 * H, prefix)
        a = ops.attention(qkv, H)
        y = ops.linear_fp8(*ops.quantize_fp8(a), oq, os_, p["bo"], h)
    close(qkv.view(B, N, 3 * H, Dh), *rotary_oracle(before.view(B, N, 3 * H, Dh), pos, freq, [8, 8], 2 * H, prefix, False), "rotary_")
    # attention of the same 16-bit q | k | v: the weights (for the second product) and the result are rounded to bf16, 2^-8 of the weights times |v| each
    z = qkv.double().view(B, N, 3, H, Dh).permute(2, 0, 3, 1, 4)
    weights = torch.softmax(z[0] @ z[1].transpose(2, 3) * Dh ** -0.5, -1)
    want, mag = ((weights @ v).transpose(1, 2).reshape(B, N, D) for v in (z[2], z[2].abs()))
    assert bool(((a.double() - want).abs() <= (2 * 2.0 ** -8 + F32) * mag).all())
    # the unquantised half in 64 bits
    pd = {k: v.double() for k, v in p.items()}
    hd = x.double() + branch.double()
    u = (norm_oracle(hd, pd["n"], 1e-6)[0] @ pd["wqkv"].t() + pd["bqkv"]).view(B, N, 3 * H, Dh)
    u = rotary_oracle(u, pos, freq, [8, 8], 2 * H, prefix, False)[0].view(B, N, 3, H, Dh).permute(2, 0, 3, 1, 4)
    out = (torch.softmax(u[0] @ u[1].transpose(2, 3) * Dh ** -0.5, -1) @ u[2]).transpose(1, 2).reshape(B, N, D) @ pd["wo"].t()
    assert float(h.double().sub(hd).norm()) <= 2.0 ** -24 * float(hd.norm())
    got = y.double() - h.double() - pd["bo"]
    assert rel(got, out) < 3 * 0.076, rel(got, out)
