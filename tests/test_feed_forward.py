"""The root-mean-square norm and the gated feed-forward block against float64 forms with derived bounds: on the GPU, and (small cases) on the CPU
stand-in build of the same kernel sources."""
import os

import pytest
import torch

import feed_forward_cases as cases
from feed_forward_cases import BF16, F16, F32

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope='module')
def emu():
    import sys
    sys.path.insert(0, HERE)
    from host_harness import standin
    from nerfool_amd import _lib
    if not os.path.exists(standin.CLANG):
        pytest.skip('no clang++ for the CPU stand-in build')
    keep = _lib._lib, _lib._emulated
    standin.install_emulated(build=True)
    yield 'cpu'
    _lib._lib, _lib._emulated = keep


NORM_SMALL = [(1, 1, F32), (1, 64, BF16), (5, 37, F32), (3, 129, F16), (9, 8, BF16), (2, 515, F32), (1, 2049, F16), (70, 20, F32)]
NORM_GPU = NORM_SMALL + [(1, 4096, BF16), (513, 64, F32), (2050, 520, BF16), (2100, 1023, F32), (2049, 4097, F16), (3, 8200, F32), (4, 16385, BF16),
                         (2, 40000, F32), (40, 70001, BF16), (32768, 64, F32), (4099, 1001, BF16)]
GATED_SMALL = [(1, 8, 8, F32), (3, 16, 24, BF16), (5, 33, 17, F16), (130, 40, 72, BF16), (2, 65, 130, F32), (17, 7, 5, BF16)]
GATED_GPU = GATED_SMALL + [(1, 1, 1, F32), (1, 256, 512, BF16), (7, 512, 300, F16), (40, 257, 129, BF16), (64, 64, 256, F32), (65, 1000, 520, F32),
                           (300, 264, 1032, BF16), (1025, 520, 260, F16), (513, 129, 65, F32), (129, 2048, 1000, BF16)]


@pytest.mark.parametrize('rows,dim,dtype', NORM_SMALL)
def test_norm_standin(emu, rows, dim, dtype):
    cases.check_norm(rows, dim, dtype, emu)


@pytest.mark.parametrize('rows,dim,hidden,dtype', GATED_SMALL)
def test_gated_standin(emu, rows, dim, hidden, dtype):
    cases.check_gated(rows, dim, hidden, dtype, emu, act=('silu', 'gelu', 'relu')[rows % 3])


@pytest.mark.gpu
@pytest.mark.parametrize('rows,dim,dtype', NORM_GPU)
def test_norm(rows, dim, dtype):
    cases.check_norm(rows, dim, dtype, 'cuda')


@pytest.mark.gpu
@pytest.mark.parametrize('residual,weight,use', [(False, True, ('y',)), (True, False, ('y', 'h')), (False, False, ('y',)), (True, True, ('y',))])
def test_norm_optional_inputs(residual, weight, use):
    cases.check_norm(37, 200, BF16, 'cuda', residual=residual, weight=weight, use=use)
    cases.check_norm(37, 8200, F32, 'cuda', residual=residual, weight=weight, use=use)


@pytest.mark.gpu
@pytest.mark.parametrize('act', ['silu', 'gelu', 'relu'])
@pytest.mark.parametrize('rows,dim,hidden,dtype', GATED_GPU)
def test_gated(rows, dim, hidden, dtype, act):
    cases.check_gated(rows, dim, hidden, dtype, 'cuda', act=act)


FROZEN_SMALL = [(70, 40, 72, F32), (130, 64, 33, BF16), (5, 17, 40, F16), (66, 7, 5, F32)]


@pytest.mark.parametrize('rows,dim,hidden,dtype', FROZEN_SMALL)
def test_gated_constant_weights_standin(emu, rows, dim, hidden, dtype):
    cases.check_gated(rows, dim, hidden, dtype, emu, act=('silu', 'gelu', 'relu')[rows % 3], frozen=True)


@pytest.mark.gpu
@pytest.mark.parametrize('act', ['silu', 'gelu', 'relu'])
@pytest.mark.parametrize('rows,dim,hidden,dtype', FROZEN_SMALL + [(1, 64, 256, F32), (4097, 64, 256, F32), (16500, 48, 700, BF16), (300, 64, 512, F16), (300, 64, 513, F32),
                                                                  (200, 65, 256, F32), (1000, 32, 100, BF16), (40000, 33, 64, F32)])
def test_gated_constant_weights(rows, dim, hidden, dtype, act):
    cases.check_gated(rows, dim, hidden, dtype, 'cuda', act=act, frozen=True)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [F32, BF16, F16])
def test_gated_large_tiles(dtype):
    """enough tiles for the largest tile form, with a ragged last tile each way"""
    cases.check_gated(2560 + 9, 1160, 2568, dtype, 'cuda', act='silu')


NORM_8BIT_SMALL = [(1, 32, BF16), (5, 37, F32), (3, 129, F16), (70, 20, F32), (1, 2049, BF16)]
GATED_8BIT_SMALL = [(1, 32, 32), (3, 64, 96), (33, 160, 32), (5, 96, 288)]


@pytest.mark.parametrize('rows,dim,dtype', NORM_8BIT_SMALL)
def test_norm_8bit_standin(emu, rows, dim, dtype):
    cases.check_norm_8bit(rows, dim, dtype, emu)
    cases.check_quantize(rows, dim, dtype, emu)


@pytest.mark.parametrize('rows,dim,hidden', GATED_8BIT_SMALL)
def test_gated_8bit_standin(emu, rows, dim, hidden):
    cases.check_gated_8bit(rows, dim, hidden, emu, act=('silu', 'gelu', 'relu')[rows % 3])


@pytest.mark.gpu
@pytest.mark.parametrize('rows,dim,dtype', NORM_8BIT_SMALL + [(16, 5120, BF16), (2100, 1023, F32), (2049, 4097, F16), (2, 40000, F32), (513, 64, F32)])
def test_norm_8bit(rows, dim, dtype):
    cases.check_norm_8bit(rows, dim, dtype, 'cuda')
    cases.check_norm_8bit(rows, dim, dtype, 'cuda', residual=False)
    cases.check_quantize(rows, dim, dtype, 'cuda')


@pytest.mark.gpu
@pytest.mark.parametrize('act,dtype', [('silu', BF16), ('gelu', F32), ('relu', F16)])
@pytest.mark.parametrize('rows,dim,hidden', GATED_8BIT_SMALL + [(1, 4096, 1024), (16, 256, 512), (129, 1056, 544), (700, 320, 2080), (2569, 1184, 2592)])
def test_gated_8bit(rows, dim, hidden, act, dtype):
    cases.check_gated_8bit(rows, dim, hidden, 'cuda', act=act, dtype=dtype)


# ---- refusals and the forms of a call: on the CPU first ------------------------------------------------------------------------------
def test_refusals(emu):
    from nerfool_amd.gnt import feed_forward as ff
    x, w = torch.zeros(4, 32), torch.zeros(32)
    ws = [torch.zeros(16, 32), torch.zeros(16, 32), torch.zeros(32, 16)]
    with pytest.raises(TypeError, match='float32, bfloat16 or float16'):
        ff.rms_norm(x.double())
    with pytest.raises(TypeError, match='weight is torch.float32'):
        ff.rms_norm(x.to(BF16), w)
    with pytest.raises(ValueError, match='weight has the shape'):
        ff.rms_norm(x, torch.zeros(31))
    with pytest.raises(ValueError, match='residual has the shape'):
        ff.rms_norm(x, w, torch.zeros(1, 32))
    with pytest.raises(ValueError, match='residual has the shape'):
        ff.rms_norm_8bit(x, w, torch.zeros(1, 32))
    with pytest.raises(ValueError, match='last axis'):
        ff.rms_norm(torch.zeros(4, 0))
    with pytest.raises(ValueError, match='last axis'):
        ff.gated_feed_forward(torch.zeros(()), *ws)
    with pytest.raises(ValueError, match='activation'):
        ff.gated_feed_forward(x, *ws, activation='tanh')
    with pytest.raises(ValueError, match='activation'):
        ff.GatedFeedForward(8, 16, 'tanh')
    with pytest.raises(ValueError, match='w_gate has the shape'):
        ff.gated_feed_forward(x, torch.zeros(16, 31), ws[1], ws[2])
    with pytest.raises(ValueError, match='w_up has the shape'):
        ff.gated_feed_forward(x, ws[0], torch.zeros(15, 32), ws[2])
    with pytest.raises(ValueError, match='w_down has the shape'):
        ff.gated_feed_forward(x, ws[0], ws[1], torch.zeros(16, 32))
    with pytest.raises(TypeError, match='w_up is torch.float16'):
        ff.gated_feed_forward(x, ws[0], ws[1].half(), ws[2])
    with pytest.raises(RuntimeError, match='no backward pass'):
        ff.rms_norm_8bit(x.requires_grad_(True), w)
    with pytest.raises(RuntimeError, match='no backward pass'):
        ff.quantize_8bit(x)
    x = x.detach()
    pair = ff.quantize_8bit(x)
    pairs = [ff.quantize_8bit(torch.zeros(s)) for s in ((64, 32), (64, 32), (32, 64))]
    assert ff.gated_feed_forward_8bit(pair, *pairs, dtype=F16).dtype == F16
    with pytest.raises(TypeError, match='dtype'):
        ff.gated_feed_forward_8bit(pair, *pairs, dtype=torch.float64)
    with pytest.raises(TypeError, match='float8_e4m3fn'):
        ff.gated_feed_forward_8bit((x, pair[1]), *pairs)
    with pytest.raises(ValueError, match='multiple of 32'):
        ff.gated_feed_forward_8bit(ff.quantize_8bit(torch.zeros(4, 40)), *pairs)
    with pytest.raises(ValueError, match="scales' leading axes"):
        ff.gated_feed_forward_8bit((pair[0], pair[1][:3]), *pairs)
    with pytest.raises(ValueError, match="w_up's scales"):
        ff.gated_feed_forward_8bit(pair, pairs[0], (pairs[1][0], pairs[1][1][:, :0]), pairs[2])
    with pytest.raises(ValueError, match='w_down has the shape'):
        ff.gated_feed_forward_8bit(pair, pairs[0], pairs[1], pairs[0])


def test_refusals_of_the_c_entries(emu):
    from nerfool_amd import _lib
    L = _lib.lib()
    assert L.nf_gated_ff_fwd_workspace_bytes(0, 8, 8, 0) == -1 and b'rows' in L.nf_last_error()
    assert L.nf_gated_ff_bwd_workspace_bytes(1, 8, 8, 3, 1, 1, 1) == -1
    for rows, dim, hidden, dtype, act in ((0, 8, 8, 0, 0), (1, 0, 8, 0, 0), (1, 8, 1 << 21, 0, 0), (1, 8, 8, 3, 0), (1, 8, 8, 0, 3)):
        assert L.nf_gated_ff_fwd(None, None, None, None, rows, dim, hidden, dtype, act, None, None, None, None, None) != 0
        assert L.nf_gated_ff_bwd(None, None, None, None, None, None, None, rows, dim, hidden, dtype, act, None, None, None, None, None, None) != 0
    for rows, dim, hidden, dtype, act in ((0, 32, 32, 1, 0), (1, 40, 32, 1, 0), (1, 32, 8, 1, 0), (1, 32, 32, 3, 0), (1, 32, 32, 1, -1)):
        assert L.nf_gated_ff_fwd_8bit(None, None, None, None, None, None, None, None, rows, dim, hidden, dtype, act, None, None, None) != 0
    a = torch.zeros(64).data_ptr()
    assert L.nf_rms_norm_fwd(a, None, None, 1, 0, 0, 1e-6, None, a, None, None, None, None) != 0
    assert L.nf_rms_norm_fwd(a, None, None, 1, 8, 0, 1e-6, None, None, None, None, None, None) != 0          # neither form of y
    assert L.nf_rms_norm_fwd(a, None, None, 1, 8, 0, 1e-6, None, a, a, a, None, None) != 0                   # both
    assert L.nf_rms_norm_fwd(a, a, None, 1, 8, 0, 1e-6, None, a, None, None, None, None) != 0                # no place for the sum
    assert L.nf_rms_norm_bwd(a, None, a, None, None, a, 1, 8, 0, a, a, None, None) != 0                      # dweight without a workspace
    assert L.nf_quantize_8bit(a, 1, 8, 7, a, a, None) != 0


def test_cpu_tensors_are_refused_without_the_standin(monkeypatch):
    from nerfool_amd import _lib
    from nerfool_amd.gnt import feed_forward as ff
    monkeypatch.setattr(_lib, '_emulated', False)
    x = torch.zeros(2, 32)
    for call in (lambda: ff.rms_norm(x), lambda: ff.quantize_8bit(x), lambda: ff.gated_feed_forward(x, torch.zeros(8, 32), torch.zeros(8, 32), torch.zeros(32, 8))):
        with pytest.raises(RuntimeError, match='GPU only'):
            call()


def test_gradients_of_gradients_are_refused(emu):
    from nerfool_amd.gnt import feed_forward as ff
    x = torch.randn(3, 16, requires_grad=True)
    ws = [torch.randn(s) for s in ((8, 16), (8, 16), (16, 8))]
    for out in (ff.rms_norm(x), ff.gated_feed_forward(x, *ws)):
        with pytest.raises(RuntimeError, match='no second derivative'):
            torch.autograd.grad(out.sum(), x, create_graph=True)


def test_unused_outputs_and_shared_leaves(emu):
    """only the sum used, only the norm used, the same tensor as x and residual, two backward passes into .grad"""
    from nerfool_amd.gnt import feed_forward as ff
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(5, 24, generator=gen, requires_grad=True)
    w = torch.ones(24, requires_grad=True)
    _, h = ff.rms_norm(x, w, x)
    gx, gw = torch.autograd.grad(h.sum(), (x, w))
    assert torch.equal(gx, torch.full_like(x, 2.0)) and torch.equal(gw, torch.zeros_like(w))
    y, _ = ff.rms_norm(x, w, x)
    plain = 2 * x.detach().double()
    plain.requires_grad_(True)
    want, = torch.autograd.grad((plain / torch.sqrt((plain * plain).mean(1, keepdim=True) + 1e-6)).sum(), plain)
    assert torch.allclose(torch.autograd.grad(y.sum(), x)[0].double(), 2 * want, atol=1e-5)
    r = torch.randn(5, 24, generator=gen, requires_grad=True)
    for k in (1, 2):          # x and the residual get one tensor as their gradient: neither's accumulation may reach the other
        y, h = ff.rms_norm(x, w, r)
        (y.sum() + (h * h).sum()).backward()
        if k == 1:
            once = x.grad.clone()
            r.grad.mul_(1.0)
    assert torch.allclose(x.grad, 2 * once) and torch.allclose(r.grad, 2 * once)


@pytest.mark.parametrize('check', ['layouts', 'empty', 'not_finite', 'extreme_8bit', 'differences', 'layer', 'layer_8bit'])
def test_forms_standin(emu, check):
    getattr(cases, 'check_' + check)(emu)


@pytest.mark.gpu
@pytest.mark.parametrize('check', ['layouts', 'empty', 'not_finite', 'extreme_8bit', 'differences', 'layer', 'layer_8bit'])
def test_forms(check):
    getattr(cases, 'check_' + check)('cuda')


@pytest.mark.gpu
def test_forms_of_other_types():
    for dtype in (F32, F16):
        cases.check_layouts('cuda', dtype)
        cases.check_layer('cuda', dtype)
        cases.check_not_finite('cuda', 300, dtype)
    cases.check_not_finite('cuda', 3000, BF16)


@pytest.mark.parametrize('rows,dim,hidden,dtype', [(3, 37, 21, F32), (67, 24, 17, BF16), (130, 70, 40, F32)])
def test_nothing_behind_the_outputs_standin(emu, rows, dim, hidden, dtype):
    cases.check_guards(emu, rows, dim, hidden, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize('rows,dim,hidden,dtype', [(1, 37, 21, F32), (67, 24, 17, BF16), (333, 64, 256, F32), (300, 129, 515, F16), (700, 1000, 333, F32), (1030, 520, 776, BF16),
                                                   (2, 4100, 70, F16), (2600, 1160, 1288, BF16)])
def test_nothing_behind_the_outputs(rows, dim, hidden, dtype):
    cases.check_guards('cuda', rows, dim, hidden, dtype)


# ---- streams and graphs ------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_another_stream():
    from nerfool_amd.gnt import feed_forward as ff
    gen = torch.Generator(device='cuda').manual_seed(1)
    x = torch.randn(600, 512, generator=gen, device='cuda').to(BF16)
    ws = [(torch.randn(*s, generator=gen, device='cuda') * 0.05).to(BF16) for s in ((1024, 512), (1024, 512), (512, 1024))]
    want = ff.gated_feed_forward(ff.rms_norm(x), *ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ff.gated_feed_forward(ff.rms_norm(x), *ws)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize('rows,dtype', [(3, BF16), (50, F32), (700, BF16), (700, F32)])
def test_captured_into_a_graph(rows, dtype):
    """forward and backward in a graph, two graphs of different calls replayed in turn with other inputs and eager work between: equal to the eager calls"""
    from nerfool_amd.gnt import feed_forward as ff
    gen = torch.Generator(device='cuda').manual_seed(2)

    def rnd(*s, scale=1.0):
        return (torch.randn(*s, generator=gen, device='cuda') * scale).to(dtype)

    dim, hid = 192, 416
    ws = [rnd(*s, scale=0.08).requires_grad_(True) for s in ((hid, dim), (hid, dim), (dim, hid))]
    wn = torch.ones(dim, dtype=dtype, device='cuda').requires_grad_(True)
    pairs = [ff.quantize_8bit(w.detach()) for w in ws]
    x, r, dy = (rnd(rows, dim) for _ in range(3))
    x.requires_grad_(True)

    def train():
        y, h = ff.rms_norm(x, wn, r)
        out = ff.gated_feed_forward(y, *ws) + h
        return (out, *torch.autograd.grad(out, (x, wn, *ws), dy))

    def serve():
        with torch.no_grad():
            q, s, h = ff.rms_norm_8bit(x, wn, r)
            return ff.gated_feed_forward_8bit((q, s), *pairs, dtype=dtype), h

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            train(), serve()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for f in (train, serve):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held = f()
        graphs.append((g, held, f))
    for k in range(4):
        with torch.no_grad():
            for t in (x, r, dy):
                t.copy_(rnd(rows, dim))
        for g, held, f in (graphs if k % 2 else graphs[::-1]):
            want = [t.clone() for t in f()]
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(held, want)), k


@pytest.mark.gpu
def test_kernel_timer_sees_the_calls():
    from nerfool_amd import prof
    from nerfool_amd.gnt import feed_forward as ff
    timer = prof.KernelTimer()
    x = torch.randn(8, 64, device='cuda')
    with prof.timing(timer):
        ff.quantize_8bit(ff.rms_norm(x))
    got = timer.summary()
    assert got['nf_rms_norm_fwd']['launches'] == got['nf_quantize_8bit']['launches'] == 1
