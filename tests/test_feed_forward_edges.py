"""The feed-forward operators where a value, a layout or a mode is at the edge of what a call may be: against float64 forms, on the GPU and (small
cases) on the CPU stand-in build of the same kernel sources."""
import pytest
import torch

from feed_forward_cases import BF16, F16, F32, check_gated, near, normal, value_of
from nerfool_amd.gnt import feed_forward as ff
from oracle import feed_forward_ref as ref
from test_feed_forward import emu  # noqa: F401  (a fixture)


# ---- relu's side ----------------------------------------------------------------------------------------------------------------------
def border_inputs(gen, rows, dim, hidden, dtype, device):
    """x, w_gate with one unit a row whose exact sum is as near to zero as the type can say: the last columns of w_gate are 1, those of x the sum of the others in as many
    parts of the type as hold 22 to 24 bits of it.  What is left is about 2^-24 of the sum, as large as what float32 sums are off by or smaller"""
    parts = {F32: 1, BF16: 3, F16: 2}[dtype]
    x = torch.randn(rows, dim, generator=gen).to(dtype)
    w = (torch.randn(hidden, dim, generator=gen) * dim ** -0.5).to(dtype)
    w[:, dim - parts:] = 1.0
    rest = -(x[:, :dim - parts].double() * w[torch.arange(rows) % hidden, :dim - parts].double()).sum(1)
    for c in range(dim - parts, dim):
        x[:, c] = rest.to(dtype)
        rest = rest - x[:, c].double()
    return x.to(device), w.to(device)


def check_relu_border(device, rows, dim, hidden, dtype, frozen):
    gen = torch.Generator().manual_seed(23 + rows)
    x, wg = border_inputs(gen, rows, dim, hidden, dtype, device)
    wu, wd = (normal(gen, *s, dtype=dtype, device=device, scale=s[1] ** -0.5) for s in ((hidden, dim), (dim, hidden)))
    dy = normal(gen, rows, dim, dtype=dtype, device=device)
    g = x.double() @ wg.double().t()
    at = torch.arange(rows, device=device)
    assert (g[at, at % hidden].abs() <= 2.0 ** -20 * x.double().norm(dim=1) * wg.double().norm(dim=1)[at % hidden]).all()
    want = ref.gated(x, wg, wu, wd, 'relu', dy, dtype, sides=True)
    ws = [t.requires_grad_(not frozen) for t in (wg, wu, wd)]
    out = ff.gated_feed_forward(x.requires_grad_(True), *ws, activation='relu')
    near(out.detach(), want['out'], 'out')
    for key, got in zip(('dx', 'dw_gate', 'dw_up', 'dw_down'), torch.autograd.grad(out, [x] if frozen else [x, *ws], dy)):
        near(got, want[key], key)


RELU_SMALL = [(5, 41, 24, F32, False), (40, 40, 33, BF16, False), (70, 37, 40, F32, False), (70, 43, 40, F16, False), (70, 40, 72, F32, True), (66, 64, 33, BF16, True),
              (3, 20, 40, F16, True)]


@pytest.mark.parametrize('rows,dim,hidden,dtype,frozen', RELU_SMALL)
def test_relu_border_standin(emu, rows, dim, hidden, dtype, frozen):  # noqa: F811
    check_relu_border(emu, rows, dim, hidden, dtype, frozen)


@pytest.mark.gpu
@pytest.mark.parametrize('rows,dim,hidden,dtype,frozen', RELU_SMALL + [
    (1, 1000, 300, BF16, False), (64, 515, 130, F32, False), (1500, 500, 1333, F32, False), (700, 1160, 520, F16, False), (2569, 1160, 2568, BF16, False),
    (2569, 1160, 2568, F32, True), (4099, 64, 256, F32, True), (4099, 30, 100, F16, True)])
def test_relu_border(rows, dim, hidden, dtype, frozen):
    check_relu_border('cuda', rows, dim, hidden, dtype, frozen)


# ---- gradients that x and the residual share ----------------------------------------------------------------------------------------------
def check_shared_gradient(device):
    """leaves of any number of axes: two passes into .grad give twice the gradient, and neither leaf's .grad is the other's memory; the sum alone used, as well"""
    gen = torch.Generator().manual_seed(29)
    for shape in ((24,), (5, 24), (2, 3, 24), (2, 1, 3, 24)):
        for use_y in (True, False):
            x, r = (normal(gen, *shape, device=device).requires_grad_(True) for _ in range(2))
            c = normal(gen, *shape, device=device)
            for k in (1, 2, 3):
                y, h = ff.rms_norm(x, None, r)
                assert y.shape == h.shape == shape
                (((y if use_y else h) * c).sum() + (h * h).sum()).backward()
                if k == 1:
                    once = x.grad.clone()
                    want, = torch.autograd.grad(((ff.rms_norm(x, None, r)[0 if use_y else 1] * c).sum() + (ff.rms_norm(x, None, r)[1] ** 2).sum()), x)
                    assert torch.allclose(once, want, rtol=2.0 ** -20, atol=2.0 ** -20)
                assert x.grad.data_ptr() != r.grad.data_ptr()
                # the passes are the same pass: k sums of one value, a rounding each
                assert torch.allclose(x.grad, k * once, rtol=k * 2.0 ** -23, atol=0) and torch.equal(x.grad, r.grad)


def test_shared_gradient_standin(emu):  # noqa: F811
    check_shared_gradient(emu)


@pytest.mark.gpu
def test_shared_gradient():
    check_shared_gradient('cuda')


# ---- calls that are no part of a gradient ---------------------------------------------------------------------------------------------------
class no_requirement:
    """nothing requires a gradient"""
    def __enter__(self):
        return self

    def __exit__(self, *_):
        return False


def check_nothing_kept(device, monkeypatch, rows, dim, hidden, dtype):
    """modules (whose weights are Parameters) under no_grad and inference_mode, and constant weights under neither: the forward without what a backward pass reads"""
    from nerfool_amd import ops
    kept = []
    gated, norm = ops.gated_ff_fwd, ops.rms_norm_fwd
    monkeypatch.setattr(ops, 'gated_ff_fwd', lambda *a, save=False: (kept.append(save), gated(*a, save=save))[1])
    monkeypatch.setattr(ops, 'rms_norm_fwd', lambda *a, want_rstd=False, **k: (kept.append(want_rstd), norm(*a, want_rstd=want_rstd, **k))[1])
    gen = torch.Generator().manual_seed(31)
    torch.manual_seed(5)
    block, rms = ff.GatedFeedForward(dim, hidden, 'gelu').to(device).to(dtype), ff.RMSNorm(dim).to(device).to(dtype)
    x, r = (normal(gen, rows, dim, dtype=dtype, device=device) for _ in range(2))
    ws = [m.weight.detach() for m in (block.gate, block.up, block.down)]
    with torch.no_grad():
        want = ref.norm(x, rms.weight, r, 1e-6, dtype=dtype)
    for mode in (torch.no_grad, torch.inference_mode, no_requirement):
        with mode():
            if mode is no_requirement:
                block.requires_grad_(False), rms.requires_grad_(False)
            y, h = rms(x, r)
            out = block(y)
            assert not out.requires_grad and not h.requires_grad and out.shape == x.shape
            near(y, want['y'], 'y'), near(h, want['h'], 'h')
            near(out, ref.gated(y, *ws, 'gelu', dtype=dtype)['out'], 'out')
            assert rms(x).shape == x.shape
    assert kept == [False] * 9
    kept.clear()
    block.requires_grad_(True)
    block(rms(x)).float().sum().backward()
    assert kept == [False, True] and block.gate.weight.grad is not None


@pytest.mark.parametrize('rows,dim,hidden,dtype', [(70, 40, 33, F32), (3, 40, 33, BF16)])
def test_nothing_kept_standin(emu, monkeypatch, rows, dim, hidden, dtype):  # noqa: F811
    check_nothing_kept(emu, monkeypatch, rows, dim, hidden, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize('rows,dim,hidden,dtype', [(70, 40, 33, F32), (3, 40, 33, BF16), (300, 64, 256, F32), (1100, 520, 264, F16), (4100, 1160, 1288, BF16)])
def test_nothing_kept(monkeypatch, rows, dim, hidden, dtype):
    check_nothing_kept('cuda', monkeypatch, rows, dim, hidden, dtype)


def test_forward_mode_is_refused(emu):  # noqa: F811
    from torch.autograd import forward_ad
    x = torch.randn(3, 16)
    ws = [torch.randn(s) for s in ((8, 16), (8, 16), (16, 8))]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for f in (lambda t: ff.rms_norm(t), lambda t: ff.gated_feed_forward(t, *ws)):
            with pytest.raises((RuntimeError, NotImplementedError)):
                f(dual)
            with torch.no_grad():
                f(x)


def test_8bit_block_refuses_a_gradient(emu):  # noqa: F811
    """a float8 tensor can require a gradient, and the block has none to give"""
    pairs = [ff.quantize_8bit(torch.ones(s)) for s in ((4, 32), (64, 32), (64, 32), (32, 64))]
    for i in range(4):
        leaf = [(q.clone().requires_grad_(True), s) if j == i else (q, s) for j, (q, s) in enumerate(pairs)]
        with pytest.raises(RuntimeError, match='gated_feed_forward_8bit has no backward pass'):
            ff.gated_feed_forward_8bit(*leaf)
        with torch.no_grad():
            assert torch.equal(ff.gated_feed_forward_8bit(*leaf), ff.gated_feed_forward_8bit(*pairs))


# ---- the norm's gradients are those of x + r, not of h as rounded to 16 bits ------------------------------------------------------------------
def check_norm_from_the_sum(device, rows, dim, dtype):
    """dy along xhat, where dx is a small difference of large values, and in the first column one sum x + r that a rounding moves by nearly half a step, for all rows alike; the
    weight a constant (as in an attack) and not: the same dx"""
    gen = torch.Generator().manual_seed(37 + rows)
    x, r = (normal(gen, rows, dim, dtype=dtype, device=device) for _ in range(2))
    eps = torch.finfo(dtype).eps
    x[:, 0], r[:, 0] = 1.0, 0.4375 * eps
    w = (1 + 0.2 * torch.randn(dim, generator=gen)).to(dtype).to(device)
    h = x.double() + r.double()
    xhat = h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-5)
    dy = (xhat / w.double()).to(dtype)
    dh = torch.zeros_like(dy)
    want = ref.norm(x, w, r, 1e-5, dy, dh, dtype, lost=0.0)
    got = []
    for trained in (False, True):
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, r)] + [w.detach().clone().requires_grad_(trained)]
        y, _ = ff.rms_norm(leaves[0], leaves[2], leaves[1], eps=1e-5)
        got.append(torch.autograd.grad(y, leaves if trained else leaves[:2], dy))
    near(got[0][0], want['dx'], 'dx, constant weight'), near(got[1][0], want['dx'], 'dx')
    near(got[1][2], want['dweight'], 'dweight')
    assert torch.equal(got[0][0], got[1][0])
    # the bound is close enough to tell: dx of h as rounded is outside of it
    assert ((ref.norm(h.to(dtype), w, None, 1e-5, dy, None, dtype)['dx'][0] - want['dx'][0]).abs() > want['dx'][1]).any()


def check_dweight_from_the_sum(device, rows, dim, dtype):
    """half of the columns hold sums that a rounding to the type moves by 7 / 16 of a step, all the same way: with the rounding of dweight itself some of them come out beyond
    its half step if they are made from h as rounded"""
    gen = torch.Generator().manual_seed(41 + rows)
    x, r = (normal(gen, rows, dim, dtype=dtype, device=device) for _ in range(2))
    eps = torch.finfo(dtype).eps
    x[:, ::2] = (1 + eps * torch.arange((dim + 1) // 2).remainder(100)).to(dtype).to(device)
    r[:, ::2] = 0.4375 * eps
    w = torch.ones(dim, dtype=dtype, device=device).requires_grad_(True)
    dy = torch.ones_like(x)
    want = ref.norm(x, w.detach(), r, 1e-5, dy, torch.zeros_like(dy), dtype, lost=0.0)['dweight']
    got, = torch.autograd.grad(ff.rms_norm(x, w, r, eps=1e-5)[0], w, dy)
    near(got, want, 'dweight')
    lost = ref.norm((x.double() + r.double()).to(dtype), w.detach(), None, 1e-5, dy, None, dtype)['dweight'][0]
    assert ((lost.to(dtype).double() - want[0]).abs() > want[1]).any()


SUMS_SMALL = [(1, 64, BF16), (9, 520, BF16), (3, 129, F16), (40, 24, BF16)]


@pytest.mark.parametrize('rows,dim,dtype', SUMS_SMALL)
def test_norm_from_the_sum_standin(emu, rows, dim, dtype):  # noqa: F811
    check_norm_from_the_sum(emu, rows, dim, dtype)
    check_dweight_from_the_sum(emu, rows, dim, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize('rows,dim,dtype', SUMS_SMALL + [(513, 520, BF16), (300, 4100, F16), (3, 40000, BF16)])
def test_norm_from_the_sum(rows, dim, dtype):
    check_norm_from_the_sum('cuda', rows, dim, dtype)
    check_dweight_from_the_sum('cuda', rows, dim, dtype)


# ---- float16 gradients without a loss scale ------------------------------------------------------------------------------------------------------
def check_small_gradients(device, rows, dim, hidden, frozen, size):
    """dy of `size`: dg and du have to be held as well as those of a larger dy, whatever the results are rounded to.  Where all rows are alike in size, of the power of two
    that brings the largest |dy| to 2^-4, half of it (a row's own largest may decide)"""
    gen = torch.Generator().manual_seed(43 + rows)
    x = normal(gen, rows, dim, dtype=F16, device=device).requires_grad_(True)
    ws = [normal(gen, *s, dtype=F16, device=device, scale=s[1] ** -0.5).requires_grad_(not frozen) for s in ((hidden, dim), (hidden, dim), (dim, hidden))]
    dy = normal(gen, rows, dim, dtype=F16, device=device, scale=size)
    for dy in (dy, dy * 2.0 ** 6):
        want = ref.gated(x.detach(), *(w.detach() for w in ws), 'silu', dy, F16, scale=max(1.0, 2.0 ** -5 / float(dy.abs().max())))
        for key, g in zip(('dx', 'dw_gate', 'dw_up', 'dw_down'), torch.autograd.grad(ff.gated_feed_forward(x, *ws), [x] if frozen else [x, *ws], dy)):
            near(g, want[key], key)


SMALL_DY = [(70, 72, 40, False, 1e-5), (130, 80, 24, False, 2e-6), (70, 40, 72, True, 1e-5), (20, 24, 40, True, 1e-6), (5, 72, 33, False, 1e-4), (66, 72, 33, False, 10.0)]


@pytest.mark.parametrize('rows,dim,hidden,frozen,size', SMALL_DY)
def test_small_gradients_standin(emu, rows, dim, hidden, frozen, size):  # noqa: F811
    check_small_gradients(emu, rows, dim, hidden, frozen, size)


@pytest.mark.gpu
@pytest.mark.parametrize('rows,dim,hidden,frozen,size', SMALL_DY + [(1025, 520, 260, False, 1e-5), (2569, 1160, 1288, False, 1e-5), (4097, 64, 256, True, 1e-5)])
def test_small_gradients(rows, dim, hidden, frozen, size):
    check_small_gradients('cuda', rows, dim, hidden, frozen, size)


def test_8bit_workspace_refuses_sizes(emu):  # noqa: F811
    from nerfool_amd import _lib
    L = _lib.lib()
    for rows, dim, hidden in ((0, 32, 32), (-5, 32, 64), (2 ** 31, 32, 32), (1, 40, 32), (1, 32, 8), (1, 0, 32), (1, 32, 2 ** 21)):
        assert L.nf_gated_ff_fwd_8bit_workspace_bytes(rows, dim, hidden) == -1, (rows, dim, hidden)
        assert b'nf_gated_ff_fwd_8bit_workspace_bytes' in L.nf_last_error()
    assert L.nf_gated_ff_fwd_8bit_workspace_bytes(1, 32, 32) > 0


# ---- the 8-bit block's tiles --------------------------------------------------------------------------------------------------------------------
def pair_of(values, scale_bytes):
    return values.to(torch.float8_e4m3fn), scale_bytes.to(torch.uint8).view(torch.float8_e8m0fnu)


def check_8bit_exact_products(device, rows, dim, hidden, dtype):
    """operands whose products lose nothing on any instruction, so that the bound is that of one rounding: of 16 consecutive k one x and one w_down is not zero.  g and u are exact:
    products are multiples of 2^-4 up to 2^5, dim / 16 of them below 2^15 in all, so h is the float32 product of two known values and its 8-bit form is known; out is a float32
    sum of hidden / 16 products.  Every 32-block has a scale of its own"""
    gen = torch.Generator().manual_seed(47 + rows + dim)

    def scales(n, k, least=126):
        return torch.randint(least, least + 3, (n, k // 32), generator=gen)

    def dense(n, k):          # 1, 1.5 or 2, either sign
        return torch.randint(2, 5, (n, k), generator=gen).float() / 2 * (torch.randint(0, 2, (n, k), generator=gen) * 2 - 1)

    def sparse(n, k):         # one of 0.5, 1, 2 in 16
        v = torch.zeros(n, k // 16, 16)
        v.scatter_(2, torch.randint(0, 16, (n, k // 16, 1), generator=gen), torch.exp2(torch.randint(-1, 2, (n, k // 16, 1), generator=gen).float()) *
                   (torch.randint(0, 2, (n, k // 16, 1), generator=gen) * 2 - 1))
        return v.view(n, k)

    # (w_down times 2^-9: float16 results stay in its range)
    pairs = [pair_of(make(n, k).to(device), scales(n, k, least).to(device)) for make, n, k, least in
             ((sparse, rows, dim, 126), (dense, hidden, dim, 126), (dense, hidden, dim, 126), (sparse, dim, hidden, 117))]
    out = ff.gated_feed_forward_8bit(*pairs, activation='relu', dtype=dtype)
    x, wg, wu, wd = (value_of(*p) for p in pairs)
    g, u = x @ wg.t(), x @ wu.t()
    assert (dim // 16) * 2.0 ** 5 < 2.0 ** 15 and float(g.abs().max()) < 2.0 ** 15 and torch.equal(g * 16, torch.round(g * 16))
    h = (g.clamp(min=0).float() * u.float()).double()
    hq, s = ref.to_8bit(h)
    hq = hq * s.repeat_interleave(32, dim=1)
    near(out, (hq @ wd.t(), ref.rounded(hq @ wd.t(), (hidden // 16 + 8) * 2.0 ** -23 * (hq.abs() @ wd.abs().t()), dtype)), 'out')


def check_8bit_norm(device, rows, dim, hidden, act):
    """the bfloat16 form as a whole, where bounds of single values are too wide to tell: the relative distance from the float64 form.  Rounding the result: at most 2^-9.  The scaled
    instruction drops of each product what lies below 2^-12 of the largest of 16, which is some 3.5 times their rms: 16 of them are off by at most 4 * 2^-12 * 3.5 of the rms of a
    product, and lost in a sum of K / 16 such groups 2^-12 * 3.5 / 4 * 4 / 4 ~ 2^-12 of the sum's; g and u together 2^-11.5.  A value of h that is off by 2^-11.5 of itself takes the
    neighbouring step (2^-3 of itself at most, 2^-4 at least) for one in 2^7.5, which is 2^-3 * 2^-3.75 = 2^-6.75 of h and of out"""
    gen = torch.Generator().manual_seed(53 + rows)
    pairs = [ff.quantize_8bit(normal(gen, *s, device=device, scale=c)) for s, c in
             (((rows, dim), 1.0), ((hidden, dim), dim ** -0.5), ((hidden, dim), dim ** -0.5), ((dim, hidden), hidden ** -0.5))]
    out = ff.gated_feed_forward_8bit(*pairs, activation=act, dtype=BF16).double()
    x, wg, wu, wd = (value_of(*p) for p in pairs)
    hq, s = ref.to_8bit(ref.act(act, x @ wg.t())[0] * (x @ wu.t()))
    want = (hq * s.repeat_interleave(32, dim=1)) @ wd.t()
    assert float((out - want).norm() / want.norm()) <= (2.0 ** -18 + 2.0 ** -13.5) ** 0.5


TILES_8BIT_SMALL = [(70, 96, 160), (65, 32, 64), (130, 160, 32)]          # (k off the step of 128 by 32, 64 and 96)
# (4100 x 2592 from 288: enough tiles for the 256 x 256 form of the down product, 2569 x 2592 from 1184 of the gated one)
TILES_8BIT = TILES_8BIT_SMALL + [(129, 1056, 544), (700, 320, 2080), (300, 4096, 128), (2569, 1184, 2592), (4100, 2592, 288), (64, 96, 160)]


@pytest.mark.parametrize('rows,dim,hidden', TILES_8BIT_SMALL)
def test_8bit_tiles_standin(emu, rows, dim, hidden):  # noqa: F811
    for dtype in (BF16, F32):
        check_8bit_exact_products(emu, rows, dim, hidden, dtype)
    check_8bit_norm(emu, rows, dim, hidden, 'silu')


@pytest.mark.gpu
@pytest.mark.parametrize('rows,dim,hidden', TILES_8BIT)
def test_8bit_tiles(rows, dim, hidden):
    for dtype in (BF16, F32, F16):
        check_8bit_exact_products('cuda', rows, dim, hidden, dtype)
    for act in ('silu', 'gelu', 'relu'):
        check_8bit_norm('cuda', rows, dim, hidden, act)


# ---- every form of the largest tile ---------------------------------------------------------------------------------------------------------------
GATE_UP, DOWN, DH, DX, DW_GATE_UP, DW_DOWN = range(6)
# sizes, ragged each way, and the products that take 256 x 256 tiles there, with the sum in one part or in several
LARGE = [((2569, 520, 4104), {GATE_UP: 1, DOWN: 7, DH: 1, DX: 7, DW_GATE_UP: 2}), ((4105, 2053, 264), {DOWN: 1, DX: 1}),
         ((521, 2053, 4104), {DW_GATE_UP: 1, DW_DOWN: 1}), ((4105, 520, 2568), {GATE_UP: 1, DH: 1, DX: 5, DW_GATE_UP: 4, DW_DOWN: 7})]


def form(rows, dim, hidden, dtype, product):
    from nerfool_amd import _lib
    f = _lib.lib().nf_gated_ff_form(rows, dim, hidden, {F32: 0, BF16: 1, F16: 2}[dtype], product)
    return f & 0xffff, f >> 16


def test_large_tiles_cover_every_form(emu):  # noqa: F811
    for dtype in (BF16, F16):
        reached = set()
        for sizes, products in LARGE:
            for product, parts in products.items():
                assert form(*sizes, dtype, product) == (256, parts), (sizes, product)
                reached.add((product, parts > 1))
        assert reached == {(GATE_UP, False), (DH, False)} | {(p, split) for p in (DOWN, DX, DW_GATE_UP, DW_DOWN) for split in (False, True)}
    assert form(64, 520, 4104, BF16, DOWN) == (0, 0) and form(64, 520, 4104, F32, DX)[0] == 128
    from nerfool_amd import _lib
    L = _lib.lib()
    assert L.nf_gated_ff_8bit_form(4100, 2592, 288, 1) == L.nf_gated_ff_8bit_form(2569, 1184, 2592, 0) == 1 << 16 | 256
    assert L.nf_gated_ff_8bit_form(64, 96, 160, 0) == 0 and L.nf_gated_ff_8bit_form(65, 96, 160, 0) == 1 << 16 | 128
    for bad in ((0, 8, 8, 0, 0), (1, 8, 8, 3, 0), (1, 8, 8, 0, 6), (1, 8, 8, 0, -1)):
        assert L.nf_gated_ff_form(*bad) == -1 and b'nf_gated_ff_form' in L.nf_last_error()
    for bad in ((0, 32, 32, 0), (1, 40, 32, 0), (1, 32, 32, 2)):
        assert L.nf_gated_ff_8bit_form(*bad) == -1 and b'nf_gated_ff_8bit_form' in L.nf_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [BF16, F16])
@pytest.mark.parametrize('sizes', [s for s, _ in LARGE])
def test_large_tiles(sizes, dtype):
    check_gated(*sizes, dtype, 'cuda', act='silu')


# ---- graphs, and offsets beyond 32 bits ------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize('rows,dim,hidden,dtype,frozen', [(3, 72, 104, F16, False), (70, 192, 416, F16, False), (700, 192, 416, F32, False), (300, 64, 256, F16, True),
                                                          (300, 64, 256, F32, True)])
def test_relu_captured_into_a_graph(rows, dim, hidden, dtype, frozen):
    """what relu and float16 add to a pass (row norms, sums in double, the gradients' power of two) is made anew by each replay: dy a thousand times smaller, units on the border"""
    gen = torch.Generator().manual_seed(59)
    x, wg = border_inputs(gen, rows, dim, hidden, dtype, 'cuda')
    ws = [t.requires_grad_(not frozen) for t in (wg, *(normal(gen, *s, dtype=dtype, device='cuda', scale=s[1] ** -0.5) for s in ((hidden, dim), (dim, hidden))))]
    x.requires_grad_(True)
    dy = normal(gen, rows, dim, dtype=dtype, device='cuda')

    def train():
        out = ff.gated_feed_forward(x, *ws, activation='relu')
        return (out, *torch.autograd.grad(out, [x] if frozen else [x, *ws], dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            train()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = train()
    for k in range(4):
        fresh, other = border_inputs(gen, rows, dim, hidden, dtype, 'cuda')
        with torch.no_grad():
            x.copy_(fresh), wg.copy_(other), dy.copy_(normal(gen, rows, dim, device='cuda', scale=1000.0 ** -(k % 2)))
        want = [t.clone() for t in train()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), k


def ends(rows, n=40):
    return torch.cat([torch.arange(n), torch.arange(rows - n, rows)]).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize('rows,dim,hidden,dtype,frozen,act', [(262300, 72, 8200, BF16, False, 'relu'), ((1 << 25) + 77, 64, 40, BF16, True, 'gelu')])
def test_gated_offsets_beyond_32_bits(rows, dim, hidden, dtype, frozen, act):
    """rows x hidden, or rows x dim, above 2^31 values: the first and the last rows"""
    gen = torch.Generator(device='cuda').manual_seed(61)
    x = torch.randn(rows, dim, generator=gen, device='cuda', dtype=dtype).requires_grad_(True)
    dy = torch.randn(rows, dim, generator=gen, device='cuda', dtype=dtype)
    ws = [(torch.randn(*s, generator=gen, device='cuda') * s[1] ** -0.5).to(dtype).requires_grad_(not frozen) for s in ((hidden, dim), (hidden, dim), (dim, hidden))]
    out = ff.gated_feed_forward(x, *ws, activation=act)
    grads = torch.autograd.grad(out, [x] if frozen else [x, *ws], dy)
    at = ends(rows)
    want = ref.gated(x.detach()[at], *(w.detach() for w in ws), act, dy[at], dtype, sides=True)
    near(out.detach()[at], want['out'], 'out'), near(grads[0][at], want['dx'], 'dx')
    if not frozen:          # the gradients of the weights are linear in dy: of the ends alone, the rest zero
        dy.zero_()[at] = torch.randn(len(at), dim, generator=gen, device='cuda', dtype=dtype)
        want = ref.gated(x.detach()[at], *(w.detach() for w in ws), act, dy[at], dtype, sides=True)
        for key, got in zip(('dw_gate', 'dw_up', 'dw_down'), torch.autograd.grad(ff.gated_feed_forward(x, *ws, activation=act), ws, dy)):
            near(got, want[key], key)


@pytest.mark.gpu
def test_norm_and_8bit_offsets_beyond_32_bits():
    rows, dim = (1 << 20) + 77, 2080
    gen = torch.Generator(device='cuda').manual_seed(67)
    x, r, dy = (torch.randn(rows, dim, generator=gen, device='cuda', dtype=BF16) for _ in range(3))
    at = ends(rows)
    x.requires_grad_(True)
    y, h = ff.rms_norm(x, None, r)
    want = ref.norm(x.detach()[at], None, r[at], 1e-6, dy[at], torch.zeros_like(dy[at]), BF16, lost=0.0)
    near(y.detach()[at], want['y'], 'y'), near(h.detach()[at], want['h'], 'h')
    near(torch.autograd.grad(y, x, dy)[0][at], want['dx'], 'dx')
    del y, h, dy
    x = x.detach()
    q, s, _ = ff.rms_norm_8bit(x, None, r)
    small = ff.rms_norm_8bit(x[at], None, r[at])
    assert torch.equal(q[at].view(torch.uint8), small[0].view(torch.uint8)) and torch.equal(s[at].view(torch.uint8), small[1].view(torch.uint8))
    pairs = [ff.quantize_8bit(torch.randn(*n, generator=gen, device='cuda') * 0.02) for n in ((64, dim), (64, dim), (dim, 64))]
    out = ff.gated_feed_forward_8bit((q, s), *pairs, dtype=BF16)
    # (fewer rows may take another form, whose sums are in another order: the bound of check_8bit_norm)
    small = ff.gated_feed_forward_8bit((q[torch.cat([at] * 4)], s[torch.cat([at] * 4)]), *pairs, dtype=BF16)[:len(at)].double()
    assert float((out[at].double() - small).norm() / small.norm()) <= (2.0 ** -18 + 2.0 ** -13.5) ** 0.5


def check_relu_zeros(device, rows, dim, hidden, dtype, frozen):
    """rows of zeros, and gate rows of zeros: g is 0 exactly, and so is relu's slope there"""
    gen = torch.Generator().manual_seed(71)
    x = normal(gen, rows, dim, dtype=dtype, device=device)
    ws = [normal(gen, *s, dtype=dtype, device=device, scale=s[1] ** -0.5) for s in ((hidden, dim), (hidden, dim), (dim, hidden))]
    x[::3], ws[0][::2] = 0, 0
    dy = normal(gen, rows, dim, dtype=dtype, device=device)
    want = ref.gated(x, *ws, 'relu', dy, dtype, sides=True)
    ws = [w.requires_grad_(not frozen) for w in ws]
    out = ff.gated_feed_forward(x.requires_grad_(True), *ws, activation='relu')
    grads = torch.autograd.grad(out, [x] if frozen else [x, *ws], dy)
    near(out.detach(), want['out'], 'out')
    for key, got in zip(('dx', 'dw_gate', 'dw_up', 'dw_down'), grads):
        near(got, want[key], key)
    assert (grads[0][::3] == 0).all() and (frozen or (grads[1][::2] == 0).all())


ZEROS = [(5, 41, 24, F32, False), (70, 37, 40, BF16, False), (70, 40, 33, F32, True), (66, 64, 50, F16, True)]


@pytest.mark.parametrize('rows,dim,hidden,dtype,frozen', ZEROS)
def test_relu_zeros_standin(emu, rows, dim, hidden, dtype, frozen):  # noqa: F811
    check_relu_zeros(emu, rows, dim, hidden, dtype, frozen)


@pytest.mark.gpu
@pytest.mark.parametrize('rows,dim,hidden,dtype,frozen', ZEROS + [(700, 200, 300, F32, False), (1300, 64, 257, F32, True)])
def test_relu_zeros(rows, dim, hidden, dtype, frozen):
    check_relu_zeros('cuda', rows, dim, hidden, dtype, frozen)
