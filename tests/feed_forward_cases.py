"""Cases of the feed-forward operators, run by test_feed_forward.py on the GPU and on the CPU stand-in build of the kernels."""
import torch

from nerfool_amd.gnt import feed_forward as ff
from oracle import feed_forward_ref as ref

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def near(got, want, what):
    value, bound = want
    assert torch.isfinite(got.double()).all(), what
    off = (got.double() - value).abs()
    worst = (off / bound.clamp(min=1e-300)).max() if off.numel() else 0.0
    assert (off <= bound).all(), '%s: off by %.3g of its bound' % (what, float(worst))


def normal(gen, *shape, dtype=F32, device='cpu', scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(dtype).to(device)


def check_norm(rows, dim, dtype, device, residual=True, weight=True, use=('y', 'h'), seed=0):
    gen = torch.Generator().manual_seed(seed + 7 * rows + dim)
    x = normal(gen, rows, dim, dtype=dtype, device=device)
    r = normal(gen, rows, dim, dtype=dtype, device=device) if residual else None
    w = (1 + 0.2 * torch.randn(dim, generator=gen)).to(dtype).to(device) if weight else None
    dy, dh = (normal(gen, rows, dim, dtype=dtype, device=device) if k in use else None for k in ('y', 'h'))
    leaves = [t for t in (x, r, w) if t is not None]
    for t in leaves:
        t.requires_grad_(True)
    got = ff.rms_norm(x, w, r, eps=1e-5)
    y, h = got if residual else (got, None)
    want = ref.norm(x.detach(), None if w is None else w.detach(), None if r is None else r.detach(), 1e-5, dy, dh if residual else None, dtype)
    near(y.detach(), want['y'], 'y')
    outs, grads = [y], [dy]
    if residual:
        near(h.detach(), want['h'], 'h')
        if 'h' in use:
            outs, grads = [y, h], [dy, dh]
    back = torch.autograd.grad(outs, leaves, grads)
    near(back[0], want['dx'], 'dx')
    if residual:
        near(back[1], want['dx'], 'dresidual')
    if weight:
        near(back[-1], want['dweight'], 'dweight')
    again = torch.autograd.grad(ff.rms_norm(x, w, r, eps=1e-5) if residual else [ff.rms_norm(x, w, r, eps=1e-5)], leaves,
                                [dy, dh if dh is not None else torch.zeros_like(dy)] if residual else grads)
    if not residual or 'h' in use:
        assert all(torch.equal(a, b) for a, b in zip(back, again)), 'the same call again'


def check_gated(rows, dim, hidden, dtype, device, act='silu', frozen=False, seed=0, scale=1.0):
    gen = torch.Generator().manual_seed(seed + rows + 3 * dim + 5 * hidden)
    x = normal(gen, rows, dim, dtype=dtype, device=device, scale=scale).requires_grad_(True)
    ws = [normal(gen, *s, dtype=dtype, device=device, scale=s[1] ** -0.5).requires_grad_(not frozen) for s in ((hidden, dim), (hidden, dim), (dim, hidden))]
    dy = normal(gen, rows, dim, dtype=dtype, device=device)
    with torch.no_grad():
        plain = ff.gated_feed_forward(x, *ws, activation=act)
    out = ff.gated_feed_forward(x, *ws, activation=act)
    want = ref.gated(x.detach(), *(w.detach() for w in ws), act, dy, dtype)
    near(plain, want['out'], 'out without a gradient')
    near(out.detach(), want['out'], 'out')
    leaves = [x] if frozen else [x, *ws]
    for key, got in zip(('dx', 'dw_gate', 'dw_up', 'dw_down'), torch.autograd.grad(out, leaves, dy)):
        near(got, want[key], key)
