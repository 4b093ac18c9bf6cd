"""Orthogonalised updates and the optimizer step built on them, against the
formulas in 64 bits.

Tolerances. One step is bounded entry by entry. A product's operands are two
fp16 numbers (each value to 2^-22), the product of the two low parts (2^-22) is
left out, and at most 48 partial sums are cut off at 2^-23 of them before they
are added in fp32 (at most 2^9 parts at 2^-24): 1e-5 of the same product of
absolute values covers it. bf16 runs hold A and B, and X inside A, to fp16's
2^-11. The chain b A + c A A, then times X, holds at most 8 such errors.

After several steps the yardstick is the same formula in fp32 (torch on the
CPU): its own distance from 64 bits, times 4, plus the rounding to the result's
type (half a step: 2^-9 of a bf16 value, twice, since such a run may add as
much of its own).
"""
import importlib
import math

import pytest
import torch

gpu = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ABC = (3.4445, -4.7750, 2.0315)


def plain(u, steps=5, abc=ABC, eps=1e-7, dtype=torch.float64):
    a, b, c = abc
    x = u.detach().cpu().double()
    x = (x / torch.linalg.matrix_norm(x, keepdim=True).clamp(min=eps)).to(dtype)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    for _ in range(steps):
        g = x @ x.mT
        x = a * x + (b * g + c * g @ g) @ x
    return x.mT if tall else x


def rel(got, ref):
    return float((got.detach().double().cpu() - ref).norm() / ref.norm())


def strong(m, n, rank, dtype=F32, batch=None, seed=0, scale=1e-3):
    gen = torch.Generator().manual_seed(seed)
    lead = () if batch is None else (batch,)
    u = torch.randn(*lead, m, rank, generator=gen) @ torch.randn(*lead, rank, n, generator=gen)
    return (scale * (u + 0.05 * torch.randn(*lead, m, n, generator=gen))).to(dtype)


SIZES = [(1, 1), (1, 70), (70, 1), (16, 16), (63, 65), (64, 64), (128, 128), (129, 127), (45, 3000), (200, 130),
         (257, 255), (384, 640), (1000, 300),
         # on chip in 1, 4 and 8 blocks, and just beyond
         (100, 256), (100, 257), (512, 128), (90, 513), (128, 1024), (1000, 17), (128, 1025), (129, 1024), (60, 1500),
         (2048, 128), (33, 2049)]


@gpu
@pytest.mark.parametrize("m,n", SIZES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_one_step_entry_by_entry(gs, m, n, dtype):
    u = strong(m, n, 2, dtype)     # few directions: singular values near 1, all terms count
    for abc in (ABC, (0.0, 1.0, 0.0), (0.0, 0.0, 1.0)):
        got = gs.orthogonalize(u.to(DEV), steps=1, coefficients=abc)
        assert got.dtype == dtype and got.shape == u.shape and got.is_contiguous()
        ref = plain(u, 1, abc)
        size = plain(u.abs(), 1, tuple(abs(v) for v in abc))
        unit = 1e-5 if dtype != BF16 else 2.0 ** -11
        half = torch.finfo(dtype).eps / 2
        tol = 8 * unit * size + half * ref.abs() + torch.finfo(dtype).tiny
        err = (got.double().cpu() - ref).abs()
        assert bool((err <= tol).all()), (abc, float((err / tol).max()))


@gpu
@pytest.mark.parametrize("m,n", SIZES + [(1024, 1024), (700, 2100)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_five_steps(gs, m, n, dtype):
    u = strong(m, n, max(1, min(m, n) // 16), dtype, seed=m)
    got = gs.orthogonalize(u.to(DEV))
    ref = plain(u)
    yard = rel(plain(u, dtype=F32), ref)
    round_off = {F32: 0.0, F16: 2.0 ** -12, BF16: 2 * 2.0 ** -9}[dtype]
    assert rel(got, ref) <= 4 * yard + 2 ** -22 + round_off


@gpu
@pytest.mark.parametrize("batch,m,n,dtype", [
    (12, 256, 512, BF16), (1, 1536, 1536, BF16), (1, 2048, 4096, BF16), (1, 3001, 3501, BF16),
    (32, 384, 384, F32), (1, 1333, 1000, F32), (1, 2100, 2050, F16), (7, 130, 2300, F32)])
def test_every_tile_shape(gs, batch, m, n, dtype):
    """Sizes whose products are cut into each of the tile shapes, some of them into more
    rounds of tiles than one; the formulas run on the GPU, in 64 bits and (the yardstick) 32."""
    gen = torch.Generator(device=DEV).manual_seed(m)
    u = torch.randn(batch, m, n, generator=gen, device=DEV)
    u = (1e-3 * (u + 0.2 * torch.randn(batch, m, 8, generator=gen, device=DEV) @
                 torch.randn(batch, 8, n, generator=gen, device=DEV))).to(dtype)

    def formula(kind):
        x = u.double()
        x = (x / torch.linalg.matrix_norm(x, keepdim=True)).to(kind)
        x = x.mT if m > n else x
        for _ in range(5):
            g = x @ x.mT
            x = ABC[0] * x + (ABC[1] * g + ABC[2] * g @ g) @ x
        return (x.mT if m > n else x).double()

    ref = formula(torch.float64)
    yard = float((formula(F32) - ref).norm() / ref.norm())
    got = gs.orthogonalize(u).double()
    round_off = {F32: 0.0, F16: 2.0 ** -12, BF16: 2 * 2.0 ** -9}[dtype]
    assert float((got - ref).norm() / ref.norm()) <= 4 * yard + 2 ** -22 + round_off
    # no tile of its own may be off: 128 x 128 pieces against twice the whole's bound
    worst = 0.0
    for i in range(0, m, 128):
        for j in range(0, n, 128):
            a, b = got[:, i:i + 128, j:j + 128], ref[:, i:i + 128, j:j + 128]
            worst = max(worst, float((a - b).norm() / b.norm()))
    assert worst <= 2 * (4 * yard + 2 ** -22 + round_off)


@gpu
@pytest.mark.parametrize("m,n", [(100, 300), (64, 900), (90, 1700)])
def test_stacks_of_matrices_in_clusters(gs, m, n):
    u = strong(m, n, 5, batch=4, seed=m).to(DEV)
    whole = gs.orthogonalize(u)
    for k in range(4):
        assert torch.equal(gs.orthogonalize(u[k]), whole[k])   # the same cut, the same sums
    w, m1 = torch.zeros_like(u), torch.zeros_like(u)
    gs.muon_step(w, u, m1, 0.5, beta=0.0, nesterov=False, scale=1.0)
    assert rel(w, -0.5 * whole.double().cpu()) <= 2.0 ** -22


@gpu
def test_a_graph_of_the_old_weights_is_refused(gs):
    w = torch.randn(20, 30, device=DEV, requires_grad=True)
    loss = (w * w).sum()
    gs.muon_step(w, torch.randn(20, 30, device=DEV), torch.zeros(20, 30, device=DEV), 0.1)
    with pytest.raises(RuntimeError):
        loss.backward()


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_stacks_and_strides(gs, dtype):
    u = strong(60, 100, 4, dtype, batch=5, seed=1).to(DEV)
    whole = gs.orthogonalize(u)
    assert whole.shape == u.shape
    for k in range(5):
        # a matrix alone may be cut into other tiles: the same but for the order of sums
        assert rel(gs.orthogonalize(u[k]), whole[k].double().cpu()) <= (1e-5 if dtype == F32 else 2 * 2.0 ** -9)
    same = u.mT.contiguous().mT
    assert torch.equal(gs.orthogonalize(same), whole)
    wide = torch.randn(5, 61, 240, device=DEV).to(dtype)
    wide[:, 1:, 3:203:2] = u
    assert torch.equal(gs.orthogonalize(wide[:, 1:, 3:203:2]), whole)
    assert torch.equal(gs.orthogonalize(u[:1].expand(3, -1, -1))[2], gs.orthogonalize(u[:1].repeat(3, 1, 1))[2])
    flipped = gs.orthogonalize(u.mT)
    assert torch.equal(flipped, whole.mT)
    assert gs.orthogonalize(u[:0]).shape == (0, 60, 100)


@gpu
def test_scales_zero_and_nan(gs):
    u = strong(90, 40, 3)
    ref = gs.orthogonalize(u.to(DEV))
    for power in (-60, 60):          # squares leave fp32's range, the norm does not
        got = gs.orthogonalize((u * 2.0 ** power).to(DEV), eps=1e-30)
        assert torch.equal(got, ref)
    assert torch.equal(gs.orthogonalize(torch.zeros(90, 40, device=DEV)), torch.zeros(90, 40, device=DEV))
    small = gs.orthogonalize(torch.full((4, 4), 1e-12, device=DEV), steps=1)   # eps takes over
    assert rel(small, plain(torch.full((4, 4), 1e-12), 1)) <= 1e-5
    u[3, 4] = float("nan")
    stack = torch.stack([u, strong(90, 40, 3)]).to(DEV)
    got = gs.orthogonalize(stack)
    assert not bool(torch.isfinite(got[0]).any()) and torch.equal(got[1], ref)
    u[3, 4] = float("inf")
    assert not bool(torch.isfinite(gs.orthogonalize(u.to(DEV))).all())


@gpu
def test_singular_values_come_near_one(gs):
    u = torch.randn(96, 160, generator=torch.Generator().manual_seed(2))
    s = torch.linalg.svdvals(gs.orthogonalize(u.to(DEV)).double().cpu())
    assert float(s.max()) < 1.21 and float(s.min()) > 0.6   # the quintic's band around 1
    spikes = torch.zeros(70, 90)
    spikes[5, 7] = 3.0                                       # an entry of 1 after the norm
    got = gs.orthogonalize(spikes.to(DEV))
    assert rel(got, plain(spikes)) <= 1e-5


@gpu
@pytest.mark.parametrize("shape", [(40, 72), (72, 40), (3, 64, 128), (300, 200), (1, 1)])
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("grad_dtype", [F32, BF16])
def test_steps_of_the_optimizer(gs, shape, nesterov, grad_dtype):
    gen = torch.Generator().manual_seed(7)
    w = torch.randn(*shape, generator=gen) * 0.05
    m = torch.zeros(*shape)
    param, momentum = w.to(DEV), m.to(DEV)
    W, M = w.double(), m.double()
    lr, beta, decay = 0.02, 0.9, 0.1
    scale = math.sqrt(max(1.0, shape[-2] / shape[-1]))
    for k in range(3):
        g = strong(*shape[-2:], 3, grad_dtype, batch=shape[0] if len(shape) == 3 else None, seed=k)
        gs.muon_step(param, g.to(DEV), momentum, lr, beta=beta, nesterov=nesterov, weight_decay=decay)
        M = beta * M + (1 - beta) * g.double()
        U = beta * M + (1 - beta) * g.double() if nesterov else M
        O = plain(U)
        W = (1 - lr * decay) * W - lr * scale * O
        # fp32 momentum: half a step each of its product, its sum and its factors
        assert float((momentum.double().cpu() - M).abs().max()) <= 4 * (k + 1) * 2.0 ** -24 * float(M.abs().max())
        yard = rel(plain(U.float(), dtype=F32), plain(U.float())) + 2.0 ** -20
        err = float((param.double().cpu() - W).norm())
        assert err <= (k + 1) * (lr * scale * 8 * yard * float(O.norm()) + 4 * 2.0 ** -24 * float(W.norm()))
    again = param.clone()
    gs.muon_step(param, g.to(DEV), momentum, lr, scale=0.0)
    assert torch.equal(param, again)


@gpu
def test_the_optimizer_is_gated_on_the_status_word(gs):
    nat = importlib.import_module("3dgs_from_scratch_b200._native")
    w, g, m = (torch.randn(80, 130, device=DEV) for _ in range(3))
    kept = w.clone(), m.clone()
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert nat.query("gs_check_status", nat.stream_ptr()) == 0
    nat.call("gs_selftest_set_timeout", flag.data_ptr(), nat.stream_ptr())
    gs.muon_step(w, g, m, 0.1)
    assert nat.query("gs_check_status", nat.stream_ptr()) == nat.GS_ERR_DEVICE_TIMEOUT
    assert torch.equal(w, kept[0]) and torch.equal(m, kept[1])
    gs.muon_step(w, g, m, 0.1)
    assert nat.query("gs_check_status", nat.stream_ptr()) == 0
    assert not torch.equal(w, kept[0]) and not torch.equal(m, kept[1])


@gpu
def test_the_same_bits_every_time_from_graphs_and_streams(gs):
    u = strong(300, 500, 9).to(DEV)
    w, g, m = (strong(200, 90, 5, seed=k).to(DEV) for k in range(3))
    ref = gs.orthogonalize(u)
    assert all(torch.equal(gs.orthogonalize(u), ref) for _ in range(3))
    w1, m1 = w.clone(), m.clone()
    for _ in range(2):
        gs.muon_step(w1, g, m1, 0.1)
    w2, m2 = w.clone(), m.clone()
    graphs = []
    for _ in range(2):                # two graphs, each with its own scratch
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = gs.orthogonalize(u)
            gs.muon_step(w2, g, m2, 0.1)
        graphs.append((graph, out))
    assert torch.equal(w2, w)         # captured, not run
    for graph, out in graphs:
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref)
    assert torch.equal(w2, w1) and torch.equal(m2, m1)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(3)], []
    for s in streams:                 # calls side by side
        with torch.cuda.stream(s):
            outs.append(gs.orthogonalize(u))
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref) for o in outs)


def test_refuses_what_it_cannot_run(gs):
    x = torch.zeros(4, 6)
    for bad in (lambda: gs.orthogonalize(x), lambda: gs.orthogonalize(x[0]), lambda: gs.orthogonalize(x[:0]),
                lambda: gs.orthogonalize(x.double()), lambda: gs.orthogonalize(x[None, None]),
                lambda: gs.muon_step(x, x, x, 0.1)):
        with pytest.raises(ValueError):
            bad()


@gpu
def test_refuses_wrong_steps_and_parameters(gs):
    x = torch.ones(4, 6, device=DEV)
    for kw in (dict(steps=0), dict(steps=101), dict(steps=1.5), dict(coefficients=(1.0, 2.0)), dict(eps=0.0),
               dict(coefficients=(float("nan"), 0.0, 0.0))):
        with pytest.raises(ValueError):
            gs.orthogonalize(x, **kw)
    nat = importlib.import_module("3dgs_from_scratch_b200._native")
    with pytest.raises(nat.NativeError):
        gs.orthogonalize(x, coefficients=(9.0, 0.0, 0.0))      # would leave the range
    for args in ((x, x, x[:, :3], 0.1), (x, x[:2], x, 0.1), (x.bfloat16(), x, x, 0.1), (x, x, x.half(), 0.1),
                 (x.t(), x.t(), x.t(), 0.1), (x, x.cpu(), x, 0.1), (x, x, x.cpu(), 0.1)):
        with pytest.raises(ValueError):
            gs.muon_step(*args)
    with pytest.raises(ValueError):
        gs.muon_step(x, x, x, 0.1, beta=1.0)


@gpu
def test_refuses_tensors_that_share_memory(gs):
    whole = torch.ones(3, 4, 6, device=DEV)
    a, b, c = whole
    flat = whole.reshape(-1)
    for args in ((a, b, a), (a, a, b), (a, b, b), (a, flat[30:54].view(4, 6), c),
                 (flat[12:36].view(4, 6), c, a)):
        with pytest.raises(ValueError, match="share"):
            gs.muon_step(*args, 0.1)
    gs.muon_step(a, b, c, 0.1)  # neighbours


def test_entry_points_refuse_bad_arguments(gs):
    lib = gs.load_native()
    nat = importlib.import_module("3dgs_from_scratch_b200._native")
    bad, at = nat.GS_ERR_INVALID_ARGUMENT, 0x10000

    def run(batch=1, rows=8, cols=8, kind=0, u=at, strides=(64, 8, 1), out=at, steps=5, abc=ABC, eps=1e-7,
            scratch=at, nbytes=0):
        return lib.gs_orthogonalize(batch, rows, cols, kind, u, *strides, out, steps, *abc, eps, scratch, nbytes,
                                    None)

    for kw in (dict(batch=0), dict(batch=65536), dict(rows=0), dict(cols=0), dict(rows=(1 << 24) + 1),
               dict(rows=(1 << 15) + 1, cols=(1 << 15) + 1), dict(kind=3), dict(u=None), dict(out=None),
               dict(u=at + 2), dict(strides=(64, -8, 1)), dict(steps=0), dict(steps=101), dict(eps=0.0),
               dict(eps=float("nan")), dict(abc=(8.5, 0.0, 0.0)), dict(abc=(3.0, 3.0, 3.0)),
               dict(abc=(float("nan"), 0.0, 0.0)), dict(scratch=None), dict(scratch=at + 8)):
        assert run(**kw) == bad, kw
    assert run() == nat.GS_ERR_CAPACITY
    assert run(steps=2, abc=(3.0, 0.0, 0.0)) == bad       # 3, then 9
    assert run(steps=1, abc=(3.0, 0.0, 0.0)) == nat.GS_ERR_CAPACITY
    assert lib.gs_muon_step(1, 8, 8, 0, at, at, at, 0.1, 1.0, 1, 0.0, 1.0, 5, *ABC, 1e-7, at, 0, None) == bad
    assert lib.gs_muon_step(1, 8, 8, 0, at, at, None, 0.1, 0.9, 1, 0.0, 1.0, 5, *ABC, 1e-7, at, 0, None) == bad
    assert lib.gs_orthogonalize_scratch_bytes(0, 8, 8, 0) == 0
    one = lib.gs_orthogonalize_scratch_bytes(1, 300, 500, 0)
    assert 0 < one < lib.gs_orthogonalize_scratch_bytes(2, 300, 500, 0)


# Quintics whose steps stay below 8 in X and in b A + c A A while A passes fp16's range at 2^12
# (15.99): the second step starts from |X|_2 = 4.2, 4.7 and (a Chebyshev polynomial on [0, 7.9]) 4.68.
TOO_LARGE = [(4.5, -0.3, 0.0), (5.0, -0.3, 0.0), (5.0, -20.0 / 7.9 ** 2, 16.0 / 7.9 ** 4)]
LARGEST = (3.9, -0.2, 0.0)      # from 3.7: A reaches 13.7


def test_coefficients_under_which_the_gram_matrix_leaves_the_range_are_refused(gs):
    lib = gs.load_native()
    nat = importlib.import_module("3dgs_from_scratch_b200._native")
    at = 0x10000

    def run(steps, abc, rows=8):
        ortho = lib.gs_orthogonalize(1, rows, 300, 0, at, 0, 300, 1, at, steps, *abc, 1e-7, at, 0, None)
        muon = lib.gs_muon_step(1, rows, 300, 0, at, at, at, 0.1, 0.9, 1, 0.0, 1.0, steps, *abc, 1e-7, at, 0, None)
        assert ortho == muon
        return ortho

    for rows in (8, 200):
        for abc in TOO_LARGE:
            assert run(2, abc, rows) == nat.GS_ERR_INVALID_ARGUMENT, abc
            assert run(1, abc, rows) == nat.GS_ERR_CAPACITY, abc     # A of the only step is at most 1
        assert run(2, LARGEST, rows) == nat.GS_ERR_CAPACITY


@gpu
@pytest.mark.parametrize("m,n", [(1, 70), (60, 90), (100, 900), (300, 500)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_the_largest_values_that_are_accepted(gs, m, n, dtype):
    """One entry: X is 1, 3.7 and then 3.9 * 3.7 - 0.2 * 3.7^3 = 4.30, and sums have one term. Values
    are held to e = 2^-22 (bf16 runs: A, B and the X inside A to e = 2^-11). The first step's error is
    at most (3.9 2^-22 + 6 * 0.2 e) / 3.7, which the second multiplies by |p'| s / p = 3.7, and that
    one's own (3.9 * 3.7 * 2^-22 + 6 * 0.2 * 3.7^3 e) / 4.3: 23 * 2^-22, or 16 * 2^-11 in bf16."""
    u = torch.zeros(m, n)
    u[m // 2, n // 3] = 2.0
    got = gs.orthogonalize(u.to(DEV, dtype), steps=2, coefficients=LARGEST).double().cpu()
    ref = plain(u, 2, LARGEST)
    assert abs(float(ref.max()) - 4.2994) < 1e-4
    tol = (23 * 2.0 ** -22 if dtype != BF16 else 16 * 2.0 ** -11) + torch.finfo(dtype).eps / 2
    assert float((got - ref).abs().max()) <= tol * float(ref.max())
    assert int((got != 0).sum()) == 1


@gpu
@pytest.mark.parametrize("shape", [(1024, 2048), (100, 900), (64, 64), (5, 90, 300)])
def test_a_step_is_taken_or_skipped_as_a_whole(gs, shape):
    """Another stream records an error before, during or after the step: weights and momentum are both
    those of the step, or both untouched."""
    nat = importlib.import_module("3dgs_from_scratch_b200._native")
    gen = torch.Generator(device=DEV).manual_seed(11)
    w, g, m = (torch.randn(*shape, generator=gen, device=DEV) for _ in range(3))
    w1, m1 = w.clone(), m.clone()
    gs.muon_step(w1, g, m1, 0.1)
    error = torch.ones(1, dtype=torch.int32, device=DEV)
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    assert nat.query("gs_check_status", nat.stream_ptr()) == 0
    taken = []
    for delay in range(0, 420, 20):                 # microseconds, at about 1.9 GHz
        w2, m2 = w.clone(), m.clone()
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            torch.cuda._sleep(1 + 1900 * delay)
            nat.call("gs_status_merge", error.data_ptr(), other.cuda_stream)
        gs.muon_step(w2, g, m2, 0.1)
        torch.cuda.synchronize()
        assert nat.query("gs_check_status", nat.stream_ptr()) == nat.GS_ERR_PEER
        taken.append(torch.equal(m2, m1))
        if taken[-1]:
            assert torch.equal(w2, w1), delay
        else:
            assert torch.equal(w2, w) and torch.equal(m2, m), delay
    with torch.cuda.stream(other):                  # and before it
        nat.call("gs_status_merge", error.data_ptr(), other.cuda_stream)
    torch.cuda.synchronize()
    w2, m2 = w.clone(), m.clone()
    gs.muon_step(w2, g, m2, 0.1)
    torch.cuda.synchronize()
    assert nat.query("gs_check_status", nat.stream_ptr()) == nat.GS_ERR_PEER
    assert torch.equal(w2, w) and torch.equal(m2, m)
    assert any(taken)


@gpu
def test_very_wide_bf16_matrices(gs):
    """Rows of equal size and orthogonal signs (Walsh functions), X = c S with S S^T = n I: one step with
    (0, 1, 0) gives X / m. Held to 2^-11 are X in A, twice, and A; the result is rounded to half a step.
    Sums of 8192 elements are cut off at 2^-23 in each of 512 additions of a growing sum, and 768 of
    them added at 2^-24: below 1e-4. One sum over all of K, cut off 393,216 times, would be 1.3% low."""
    m, n = 130, 3 << 21
    k = torch.arange(256, device=DEV)
    parity = k[:, None] & k
    for shift in (4, 2, 1):
        parity = parity ^ (parity >> shift)
    signs = (1 - 2 * (parity & 1))[:m].to(BF16)
    u = (signs * 1e-3).repeat(1, n // 256)
    got = gs.orthogonalize(u, steps=1, coefficients=(0.0, 1.0, 0.0))
    ref = 1 / math.sqrt(m * n) / m
    off = (got.reshape(m, n // 256, 256).float() * signs[:, None].float()).sub_(ref).abs_().max()
    assert float(off) <= (3 * 2.0 ** -11 + 2.0 ** -8 + 1e-4) * ref


@gpu
@pytest.mark.parametrize("shape", [(64, 64), (100, 900), (5, 90, 300), (600, 700)])
def test_captured_steps_replay(gs, shape):
    """On chip, in clusters, in stacks and in tiles: two replayed steps are the two steps, and a replay
    that finds an error recorded is skipped."""
    nat = importlib.import_module("3dgs_from_scratch_b200._native")
    gen = torch.Generator(device=DEV).manual_seed(12)
    w, g, m = (torch.randn(*shape, generator=gen, device=DEV) for _ in range(3))
    w1, m1 = w.clone(), m.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        gs.muon_step(w1, g, m1, 0.1, weight_decay=0.1)
    assert torch.equal(w1, w)
    for _ in range(2):
        graph.replay()
        gs.muon_step(w, g, m, 0.1, weight_decay=0.1)
    torch.cuda.synchronize()
    assert torch.equal(w1, w) and torch.equal(m1, m)
    assert nat.query("gs_check_status", nat.stream_ptr()) == 0
    error = torch.ones(1, dtype=torch.int32, device=DEV)
    nat.call("gs_status_merge", error.data_ptr(), nat.stream_ptr())
    graph.replay()
    torch.cuda.synchronize()
    assert nat.query("gs_check_status", nat.stream_ptr()) == nat.GS_ERR_PEER
    assert torch.equal(w1, w) and torch.equal(m1, m)
