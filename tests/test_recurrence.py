"""The gated linear recurrence against its definition in 64 bits, row by row.

Tolerances. With u = 2^-24, a state is a sum of products of at most 2 n + 2
rounded operations each (n rows in its sequence: one product and one sum a
row, whatever the order in which runs of rows are joined, and one more for
each of the few levels of joining), so its error is at most
(2 n + 16) u times the same recurrence run on absolute values. The gradient's
chain has the same form, and a gate's gradient is a sum over D channels of
products of the two: (4 n + 32 + D) u times the sum of absolute values.
Rounding to the output's type adds half a step, eps / 2 of the value.
"""
import importlib

import pytest
import torch

gpu = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def walk(x, g, init, bounds, reverse):
    """h and the final states by the definition; x, g (rows, channels) in 64 bits."""
    h, final = torch.zeros_like(x), init.clone()
    for s, (a, b) in enumerate(bounds):
        state = init[s].clone()
        for t in (range(b - 1, a - 1, -1) if reverse else range(a, b)):
            state = g[t] * state + x[t]
            h[t] = state
        final[s] = state
    return h, final


def walk_back(g, dh, dfinal, init, h, bounds, reverse):
    dx, dg, dinit = torch.zeros_like(dh), torch.zeros_like(dh), torch.zeros_like(init)
    for s, (a, b) in enumerate(bounds):
        order = list(range(b - 1, a - 1, -1) if reverse else range(a, b))
        v = dfinal[s].clone()
        for k in range(len(order) - 1, -1, -1):
            t = order[k]
            dx[t] = dh[t] + v
            dg[t] = dx[t] * (h[order[k - 1]] if k else init[s])
            v = g[t] * dx[t]
        dinit[s] = v
    return dx, dg, dinit


def bounds_of(rows, sequences, offsets):
    if offsets is None:
        n = rows // sequences
        return [(s * n, (s + 1) * n) for s in range(sequences)]
    return [(offsets[s], offsets[s + 1]) for s in range(len(offsets) - 1)]


def near(name, got, ref, scale, ops, dtype):
    got, half = got.detach().double().cpu(), torch.finfo(dtype).eps / 2
    tol = 1.01 * ops * U * scale + half * (ref.abs() + ops * U * scale) + torch.finfo(dtype).tiny * half * 2
    bad = (got - ref).abs() > tol
    assert not bool(bad.any()), (f"{name}: {int(bad.sum())} of {bad.numel()} off, the first at "
                                 f"{bad.nonzero()[0].tolist()}: {got[bad][0]} and not {ref[bad][0]}")


def check(gs, rows, sequences, channels, gates, *, offsets=None, dtype=F32, gate_dtype=F32,
          reverse=False, seed=0, with_initial=True, wrap=None, low=0.5, train=True):
    gen = torch.Generator().manual_seed(seed)
    per = channels // gates
    x = torch.randn(rows, channels, generator=gen).to(dtype)
    gate = (low + (1 - low) * torch.rand(rows, gates, generator=gen))
    gate[torch.rand(rows, gates, generator=gen) < 0.05] = 0.0
    gate[torch.rand(rows, gates, generator=gen) < 0.05] *= -1.0
    gate = gate.to(gate_dtype)
    init = torch.randn(sequences, channels, generator=gen) if with_initial else None
    dh = torch.randn(rows, channels, generator=gen).to(dtype)
    dfinal = torch.randn(sequences, channels, generator=gen)
    bounds = bounds_of(rows, sequences, offsets)
    shape = (rows,) if offsets is not None or sequences == 1 and wrap != "batch" else (sequences, rows // sequences)
    on = {k: v.to(DEV) for k, v in (("x", x), ("gate", gate), ("dh", dh))}
    on = {k: v.reshape(*shape, v.shape[-1]) for k, v in on.items()}
    if wrap == "strided":  # columns of a wider tensor
        wide = torch.zeros(*shape, 2 * channels + 2 * gates, dtype=dtype, device=DEV)
        wide[..., :channels] = on["x"]
        on["x"] = wide[..., :channels]
        wide = torch.full((*shape, channels + 8), float("nan"), dtype=dtype, device=DEV)
        wide[..., 3:3 + channels] = on["dh"]
        on["dh"] = wide[..., 3:3 + channels]
    leaves = [on["x"].detach().requires_grad_(train), on["gate"].detach().requires_grad_(train)]
    if with_initial:
        leaves.append(init.to(DEV).requires_grad_(train))
    offs = None if offsets is None else torch.tensor(offsets, dtype=torch.int32, device=DEV)
    h, final = gs.gated_scan(leaves[0], leaves[1], initial=leaves[2] if with_initial else None,
                             offsets=offs, reverse=reverse)
    assert h.dtype == dtype and final.dtype == F32 and h.shape == on["x"].shape
    X, G, DH = x.double(), gate.double().repeat_interleave(per, 1), dh.double()
    I = (init if with_initial else torch.zeros(sequences, channels)).double()
    n = max([b - a for a, b in bounds], default=0)
    ops = 2 * n + 16
    H, FIN = walk(X, G, I, bounds, reverse)
    HA, FA = walk(X.abs(), G.abs(), I.abs(), bounds, reverse)
    near("h", h.reshape(rows, channels), H, HA, ops, dtype)
    near("final", final, FIN, FA, ops, F32)
    if not train:
        return
    grads = torch.autograd.grad((h, final), leaves, (on["dh"], dfinal.to(DEV)))
    DX, DG, DI = walk_back(G, DH, dfinal.double(), I, H, bounds, reverse)
    DXA, DGA, DIA = walk_back(G.abs(), DH.abs(), dfinal.double().abs(), I.abs(), HA, bounds, reverse)
    near("dx", grads[0].reshape(rows, channels), DX, DXA, ops, dtype)
    fold = lambda t: t.reshape(rows, gates, per).sum(2)  # noqa: E731
    near("dgate", grads[1].reshape(rows, gates), fold(DG), fold(DGA), 4 * n + 32 + per, gate_dtype)
    if with_initial:
        near("dinitial", grads[2], DI, DIA, ops, F32)


@gpu
@pytest.mark.parametrize("rows,sequences", [(1, 1), (7, 7), (64, 2), (129, 1), (900, 3), (1500, 1)])
@pytest.mark.parametrize("channels,gates", [(1, 1), (3, 1), (16, 16), (35, 1), (72, 72), (64, 4)])
def test_batches_of_even_sequences(gs, rows, sequences, channels, gates):
    check(gs, rows, sequences, channels, gates, seed=rows + channels)


@gpu
@pytest.mark.parametrize("dtype,gate_dtype", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("channels,gates", [(40, 40), (40, 1), (40, 5), (21, 21), (21, 7), (520, 2), (301, 1)])
@pytest.mark.parametrize("reverse", [False, True])
def test_types_and_ragged_sequences(gs, dtype, gate_dtype, channels, gates, reverse):
    # empty ones at both ends and in the middle, one row, ends inside and at the edge of chunks,
    # rows behind the last
    offsets = [0, 0, 1, 129, 129, 129, 257, 320, 321, 700, 700]
    check(gs, 713, 10, channels, gates, offsets=offsets, dtype=dtype, gate_dtype=gate_dtype,
          reverse=reverse, seed=channels)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("channels", [33, 34, 75, 513, 1025, 1282])
def test_sixteen_bit_channels_that_fill_no_vectors(gs, dtype, channels):
    check(gs, 300, 5, channels, channels, offsets=[0, 131, 131, 250, 251, 297], dtype=dtype,
          gate_dtype=dtype, reverse=channels % 2 == 0, seed=channels)
    check(gs, 96, 3, channels, channels, dtype=dtype, gate_dtype=dtype, with_initial=False, seed=channels)


@gpu
@pytest.mark.parametrize("reverse", [False, True])
def test_rows_before_the_first_sequence_and_no_rows_inside(gs, reverse):
    check(gs, 300, 2, 24, 24, offsets=[130, 135, 200], reverse=reverse)
    check(gs, 300, 3, 24, 3, offsets=[300, 300, 300, 300], reverse=reverse)
    check(gs, 5, 2, 24, 1, offsets=[2, 2, 2], reverse=reverse)


@gpu
def test_many_short_sequences(gs):
    gen = torch.Generator().manual_seed(4)
    cuts = torch.randint(0, 2000, (1499,), generator=gen).sort().values.tolist()
    check(gs, 2000, 1500, 12, 12, offsets=[0] + cuts + [2000])
    check(gs, 4096, 4096, 20, 4, train=True)  # one row each


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strided_rows(gs, dtype):
    for channels, gates in ((32, 32), (30, 3)):
        check(gs, 400, 4, channels, gates, dtype=dtype, gate_dtype=dtype, wrap="strided")
        check(gs, 400, 2, channels, gates, offsets=[0, 150, 390], dtype=dtype, wrap="strided")


@gpu
def test_no_initial_state_and_a_batch_of_one(gs):
    check(gs, 260, 2, 16, 16, with_initial=False)
    check(gs, 260, 1, 16, 2, with_initial=False, wrap="batch", reverse=True)


@gpu
def test_long_memory(gs):
    check(gs, 6000, 1, 8, 8, low=0.999, seed=2)
    check(gs, 6000, 2, 9, 1, low=0.999, seed=3, reverse=True)


@gpu
def test_other_layouts_give_the_same(gs):
    gen = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(5, 70, 24, generator=gen, device=DEV)
    g = torch.rand(5, 70, 24, generator=gen, device=DEV)
    h, final = gs.gated_scan(x, g)
    tx = x.transpose(0, 1).contiguous().transpose(0, 1)       # rows of a time-major tensor
    tg = g.mT.contiguous().mT                                  # channels apart
    h2, f2 = gs.gated_scan(tx, tg)
    assert torch.equal(h, h2) and torch.equal(final, f2)
    ge = g[..., :1].expand(-1, -1, 24)                         # a broadcast gate
    leaf = g[..., :1].clone().requires_grad_(True)
    h3, _ = gs.gated_scan(x, leaf.expand(-1, -1, 24))
    h4, _ = gs.gated_scan(x, ge.contiguous())
    assert torch.equal(h3, h4)
    shared = g[..., :1].clone().requires_grad_(True)
    h5, _ = gs.gated_scan(x, shared)
    up = torch.randn(5, 70, 24, generator=gen, device=DEV)
    (d1,), (d2,) = torch.autograd.grad(h3, leaf, up), torch.autograd.grad(h5, shared, up)
    sizes = gs.gated_scan(x.abs(), shared.detach())[0].max() * gs.gated_scan(up.abs(), shared.detach())[0].max()
    assert torch.equal(h3, h5)
    assert float((d1 - d2).detach().abs().max()) <= 2 * (4 * 70 + 32 + 24) * U * 24 * float(sizes)
    offs = torch.arange(0, 351, 70, device=DEV)                # int64 offsets of the same sequences
    h6, f6 = gs.gated_scan(x.reshape(350, 24), g.reshape(350, 24), offsets=offs)
    # Even sequences and offsets may be cut into other chunks: each is within (2 n + 16) u of the
    # recurrence on absolute values from the exact states (n = 70), so they are within twice that.
    most = 2 * (2 * 70 + 16) * U * float(gs.gated_scan(x.abs(), g)[0].max())
    assert float((h6.reshape(5, 70, 24) - h).abs().max()) <= most
    assert float((f6 - final).abs().max()) <= most
    tail = torch.randn(351 * 24, device=DEV)[1:350 * 24 + 1].reshape(350, 24)  # not at 16 bytes
    h7, _ = gs.gated_scan(tail, g.reshape(350, 24), offsets=offs)
    h8, _ = gs.gated_scan(tail.clone(), g.reshape(350, 24), offsets=offs)
    assert torch.equal(h7, h8)


@gpu
def test_a_row_at_a_time_continues_a_sequence(gs):
    gen = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(6, 40, 48, generator=gen, device=DEV)
    g = torch.rand(6, 40, 48, generator=gen, device=DEV)
    whole, end = gs.gated_scan(x, g)
    state = torch.zeros(6, 48, device=DEV)
    tol = 2 * (2 * 40 + 16) * U * float(gs.gated_scan(x.abs(), g)[0].max())
    for t in range(40):
        h, state = gs.gated_scan(x[:, t:t + 1], g[:, t:t + 1], initial=state)
        assert torch.allclose(h[:, 0], whole[:, t], rtol=0, atol=tol)
    assert torch.allclose(state, end, rtol=0, atol=tol)


@gpu
def test_nan_and_infinity_stay_in_their_sequence(gs):
    for reverse in (False, True):
        x = torch.ones(600, 16, device=DEV)
        g = torch.full((600, 16), 0.5, device=DEV)
        x[210, 3], x[100, 5], g[395, 7] = float("nan"), float("inf"), float("inf")
        x[590:], g[590:] = float("nan"), float("nan")   # behind the last sequence
        offs = torch.tensor([0, 200, 400, 590], dtype=torch.int32, device=DEV)
        x.requires_grad_(True), g.requires_grad_(True)
        h, final = gs.gated_scan(x, g, offsets=offs, reverse=reverse)
        grads = torch.autograd.grad((h, final), (x, g), (torch.ones_like(h), torch.ones_like(final)))
        whole = torch.isfinite(h)
        for s, c in ((0, 5), (1, 3), (1, 7)):
            assert not bool(whole[200 * s:200 * (s + 1), c].all()) and not bool(torch.isfinite(final[s, c]))
            whole[200 * s:200 * (s + 1), c] = True
        assert bool(whole.all()) and float(h[590:].abs().max()) == 0.0
        for d in grads:
            assert float(d[590:].abs().max()) == 0.0
            assert bool(torch.isfinite(d[:, [0, 1, 2, 4, 6]]).all())


@gpu
def test_gradients_by_differences(gs):
    gen = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(90, 6, generator=gen, device=DEV)
    g = 0.2 + 0.7 * torch.rand(90, 2, generator=gen, device=DEV)
    init = torch.randn(4, 6, generator=gen, device=DEV)
    offs = torch.tensor([0, 33, 33, 70, 88], device=DEV)
    wh = torch.randn(90, 6, generator=gen, device=DEV)
    wf = torch.randn(4, 6, generator=gen, device=DEV)

    def loss(x, g, init):
        h, final = gs.gated_scan(x, g, initial=init, offsets=offs, reverse=True)
        return (h.double() * wh).sum() + (final.double() * wf).sum()

    leaves = [t.clone().requires_grad_(True) for t in (x, g, init)]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    for k, t in enumerate((x, g, init)):
        way = torch.randn(t.shape, generator=gen, device=DEV)
        step = 2.0 ** (-9 if k == 1 else -7)
        ahead, back = [[v.clone() for v in (x, g, init)] for _ in range(2)]
        ahead[k] += step * way
        back[k] -= step * way
        slope = float(loss(*ahead) - loss(*back)) / (2 * step)
        told = float((grads[k].double() * way).sum())
        # x and initial enter linearly; the gates' third derivative is what differences leave
        assert abs(slope - told) <= (2e-2 if k == 1 else 2e-3) * (1 + abs(told)), (k, slope, told)


@gpu
def test_only_one_output_used_and_missing_gradients(gs):
    x = torch.randn(3, 50, 8, device=DEV, requires_grad=True)
    g = torch.rand(3, 50, 8, device=DEV)
    h, final = gs.gated_scan(x, g)
    (a,) = torch.autograd.grad(final.sum(), x, retain_graph=True)
    (b,) = torch.autograd.grad(h.sum(), x, retain_graph=True)
    (c,) = torch.autograd.grad(h.sum() + final.sum(), x)
    assert torch.allclose(a + b, c, rtol=1e-5, atol=1e-5)
    with torch.no_grad():
        h, final = gs.gated_scan(x, g)
    assert not h.requires_grad and not final.requires_grad


@gpu
def test_the_same_bits_every_time_and_from_a_graph(gs):
    gen = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randn(20000, 40, generator=gen, device=DEV, requires_grad=True)
    g = torch.rand(20000, 1, generator=gen, device=DEV, requires_grad=True)
    offs = torch.tensor([0, 9000, 9001, 20000], dtype=torch.int32, device=DEV)
    up = torch.randn(20000, 40, generator=gen, device=DEV)

    def step():
        h, final = gs.gated_scan(x, g, offsets=offs)
        return (h, final) + torch.autograd.grad(h, (x, g), up)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ref = [t.clone() for t in step()]
        again = step()
        assert all(torch.equal(a, b) for a, b in zip(ref, again))
        del again
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        for t in out:
            t.detach().fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(ref, out))


@gpu
def test_calls_side_by_side_on_their_own_streams(gs):
    gen = torch.Generator(device=DEV).manual_seed(8)
    x = torch.randn(3, 4000, 24, generator=gen, device=DEV)
    g = torch.rand(3, 4000, 24, generator=gen, device=DEV)
    ref = gs.gated_scan(x, g)
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(4)]:
        with torch.cuda.stream(s):
            got.append(gs.gated_scan(x, g))
    torch.cuda.synchronize()
    assert all(torch.equal(h, ref[0]) and torch.equal(f, ref[1]) for h, f in got)


@gpu
def test_a_first_call_inside_a_capture(gs):
    x = torch.randn(2, 3000, 20, device=DEV)
    g = torch.rand(2, 3000, 4, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, final = gs.gated_scan(x, g, reverse=True)
    graph.replay()
    torch.cuda.synchronize()
    again = gs.gated_scan(x, g, reverse=True)
    assert torch.equal(h, again[0]) and torch.equal(final, again[1])


@gpu
def test_twice_differentiated_is_refused(gs):
    x = torch.randn(2, 9, 4, device=DEV, requires_grad=True)
    h, _ = gs.gated_scan(x, torch.rand(2, 9, 4, device=DEV, requires_grad=True))
    (dx,) = torch.autograd.grad(h.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


@gpu
@pytest.mark.parametrize("reverse", [False, True])
def test_more_than_2_31_elements(gs, reverse):
    rows, channels, tail = 1 << 21, 1100, 50           # 2.3e9 elements
    gen = torch.Generator(device=DEV).manual_seed(9)
    x = torch.zeros(rows, channels, dtype=BF16, device=DEV)
    g = torch.rand(rows, 1, generator=gen, device=DEV)
    ends = slice(0, tail) if reverse else slice(rows - tail, rows)  # what the chain reaches last
    x[ends] = torch.randn(tail, channels, generator=gen, device=DEV).to(BF16)
    small_x, small_g = x[ends].clone().requires_grad_(True), g[ends].clone().requires_grad_(True)
    h0, f0 = gs.gated_scan(small_x, small_g, reverse=reverse)
    up = torch.randn(tail, channels, generator=gen, device=DEV).to(BF16)
    d0 = torch.autograd.grad(h0, (small_x, small_g), up)
    x.requires_grad_(True), g.requires_grad_(True)
    h, final = gs.gated_scan(x, g, reverse=reverse)
    full = torch.zeros_like(h)
    full[ends] = up
    d = torch.autograd.grad(h, (x, g), full)
    # the same rows in the same order of batches or another: fp32 sums of at most 50 rows
    near = lambda a, b, t: torch.allclose(a.float(), b.float(), rtol=torch.finfo(t).eps, atol=1e-3)  # noqa: E731
    assert near(h[ends], h0, BF16) and near(final, f0, F32) and near(d[0][ends], d0[0], BF16)
    assert near(d[1][ends], d0[1], F32)
    other = slice(tail, tail + 1000) if reverse else slice(rows - tail - 1000, rows - tail)
    assert float(h.detach()[other].abs().max()) == 0.0


@gpu
def test_offsets_that_do_not_ascend_are_reported(gs):
    """The kernels index within the buffers whatever the offsets hold (checked by reading: a
    sequence number is below the count, a row below rows); the fault is in the status word."""
    nat = importlib.import_module("3dgs_from_scratch_b200._native")
    x = torch.randn(200, 8, device=DEV)
    for offsets in ([0, 120, 60, 200], [0, 50, 201], [-3, 50, 200], [0, 2 ** 33, 200]):
        assert nat.query("gs_check_status", nat.stream_ptr()) == 0
        gs.gated_scan(x, x, offsets=torch.tensor(offsets, device=DEV))
        assert nat.query("gs_check_status", nat.stream_ptr()) == nat.GS_ERR_INVALID_ARGUMENT
        gs.gated_scan(x, x, offsets=torch.tensor([0, 60, 200], device=DEV))
        assert nat.query("gs_check_status", nat.stream_ptr()) == 0


@gpu
def test_no_rows_and_no_sequences(gs):
    x = torch.zeros(0, 6, device=DEV, requires_grad=True)
    init = torch.randn(2, 6, device=DEV, requires_grad=True)
    h, final = gs.gated_scan(x, x.detach(), initial=init, offsets=torch.zeros(3, dtype=torch.int32, device=DEV))
    assert h.shape == (0, 6) and torch.equal(final, init)
    dx, dinit = torch.autograd.grad(final.sum(), (x, init))
    assert dx.shape == (0, 6) and bool((dinit == 1).all())
    h, final = gs.gated_scan(torch.zeros(0, 5, 6, device=DEV), torch.zeros(0, 5, 2, device=DEV))
    assert h.shape == (0, 5, 6) and final.shape == (0, 6)


def test_refuses_what_it_cannot_run(gs):
    x, g = torch.zeros(4, 6), torch.zeros(4, 6)
    for bad in (lambda: gs.gated_scan(x, g),                                       # not on a GPU
                lambda: gs.gated_scan(x[0], g[0]),
                lambda: gs.gated_scan(x, g[:3]),
                lambda: gs.gated_scan(x, torch.zeros(4, 4)),                       # 4 gates, 6 channels
                lambda: gs.gated_scan(x, torch.zeros(4, 0)),
                lambda: gs.gated_scan(x.double(), g.double()),
                lambda: gs.gated_scan(x, g.half()),
                lambda: gs.gated_scan(x[None], g[None], offsets=torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(ValueError):
            bad()


@gpu
def test_refuses_wrong_states_and_offsets(gs):
    x, g = torch.zeros(4, 6, device=DEV), torch.zeros(4, 6, device=DEV)
    offs = torch.tensor([0, 2, 4], device=DEV)
    for kw in (dict(initial=torch.zeros(2, 6, device=DEV)), dict(initial=torch.zeros(1, 6)),
               dict(initial=torch.zeros(1, 6, device=DEV, dtype=torch.int32)),
               dict(offsets=offs.cpu()), dict(offsets=offs[:1]), dict(offsets=offs.float()),
               dict(offsets=offs[None])):
        with pytest.raises(ValueError):
            gs.gated_scan(x, g, **kw)


def test_entry_points_refuse_bad_arguments(gs):
    lib = gs.load_native()
    nat = importlib.import_module("3dgs_from_scratch_b200._native")
    bad, P, at = nat.GS_ERR_INVALID_ARGUMENT, None, 0x10000

    def fwd(rows=8, seqs=2, channels=8, gates=8, xt=0, gt=0, x=at, xs=8, gate=at, gst=8, init=P,
            offs=P, h=at, scratch=P, nbytes=0):
        return lib.gs_gated_scan_forward(rows, seqs, channels, gates, xt, gt, x, xs, gate, gst, init,
                                         offs, 0, h, P, P, scratch, nbytes, P)

    for kw in (dict(rows=-1), dict(rows=2 ** 31), dict(seqs=0), dict(seqs=3), dict(channels=0), dict(channels=(1 << 30) + 8), dict(gates=0),
               dict(gates=3), dict(xt=3), dict(xt=1, gt=2), dict(xt=0, gt=1), dict(x=P), dict(gate=P),
               dict(h=P), dict(x=at + 4), dict(xs=9), dict(gst=11), dict(h=at + 4), dict(init=at + 2),
               dict(offs=at + 2), dict(rows=2 ** 20)):       # many tiles and no scratch
        assert fwd(**kw) == bad, kw
    assert lib.gs_gated_scan_backward(8, 2, 8, 8, 0, 0, at, 8, at, 8, P, P, 0, P, at, 8, P, at, at, P,
                                      P, 0, P) == bad         # nothing kept by the forward
    assert lib.gs_gated_scan_saved_bytes(-1, 1, 1, 8, 8, 0, 0) == 0
    assert lib.gs_gated_scan_saved_bytes(100, 1, 1, 8, 8, 0, 0) >= 100 // 8 * 8 * 4
    assert lib.gs_gated_scan_scratch_bytes(24, 1, 1, 8, 8, 0, 0, 0) == 0
    assert lib.gs_gated_scan_scratch_bytes(1 << 20, 1, 1, 8, 8, 0, 0, 1) > 0
    assert lib.gs_gated_scan_scratch_bytes(1 << 20, 5, 0, 8, 8, 0, 0, 0) > 0


def against(gs, x, gate, init, dh, dfinal, per, dtype, gate_dtype, reverse):
    """One sequence against its definition, forward and backward; all given in the direction of the recurrence.

    Values may fall below the normal range here, where an operation is off by up to q = 2^-150 besides the
    relative half step (fp32's smallest step is 2^-149), and later gates multiply that as they multiply the
    state. A row's product, its sum and a joining that ends there are three such operations, so states are
    off by at most the recurrence on absolute values with x = 4 q (`low`) more than before (0 where the state
    is exactly 0, as products and sums of zeros are), the gradients' chain likewise (`back`), and a gate's
    gradient, a sum of products u h, by the products of the one's size and the other's error, and q a term."""
    if reverse:
        x, gate, dh = x.flip(0), gate.flip(0), dh.flip(0)
    x, gate, dh = x.to(dtype), gate.to(gate_dtype), dh.to(dtype)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, gate, init)]
    h, final = gs.gated_scan(*leaves, reverse=reverse)
    grads = torch.autograd.grad((h, final), leaves, (dh.to(DEV), dfinal.to(DEV)))
    rows, bounds = x.shape[0], [(0, x.shape[0])]
    X, G, DH = x.double(), gate.double().repeat_interleave(per, 1), dh.double()
    I, DF = init.double(), dfinal.double()
    H, FIN = walk(X, G, I, bounds, reverse)
    HA, FA = walk(X.abs(), G.abs(), I.abs(), bounds, reverse)
    DX, DG, DI = walk_back(G, DH, DF, I, H, bounds, reverse)
    DXA, DGA, DIA = walk_back(G.abs(), DH.abs(), DF.abs(), I.abs(), HA, bounds, reverse)
    assert max(float(t.detach().max()) for t in (HA, FA, DXA, DGA, DIA)) < 2.0 ** 127  # nothing overflows
    q = 2.0 ** -150
    low, low_end = walk(4 * q * (HA > 0), G.abs(), torch.zeros_like(I), bounds, reverse)
    back, low_dg, low_di = walk_back(G.abs(), 4 * q * (DXA > 0), torch.zeros_like(I), I.abs(), HA + low,
                                     bounds, reverse)       # low_dg: the chain's error times |h|
    low_dg = low_dg + walk_back(G.abs(), DH.abs(), DF.abs(), torch.zeros_like(I), low, bounds, reverse)[1] + 4 * q
    fold = lambda t: t.reshape(rows, -1, per).sum(2)  # noqa: E731

    def close(name, got, ref, scale, floor, ops, kind):
        got, half = got.detach().double().cpu(), torch.finfo(kind).eps / 2
        tol = (1 + half) * (1.01 * ops * U * scale + 1.01 * floor) + half * ref.abs() + torch.finfo(kind).tiny * half * 2
        bad = ~((got - ref).abs() <= tol)
        assert not bool(bad.any()), (f"{name}: {int(bad.sum())} of {bad.numel()} off, the first at "
                                     f"{bad.nonzero()[0].tolist()}: {got[bad][0]} and not {ref[bad][0]}")

    ops = 2 * rows + 16
    close("h", h, H, HA, low, ops, dtype)
    close("final", final, FIN, FA, low_end, ops, F32)
    close("dx", grads[0], DX, DXA, back, ops, dtype)
    close("dgate", grads[1], fold(DG), fold(DGA), fold(low_dg), 4 * rows + 32 + per, gate_dtype)
    close("dinitial", grads[2], DI, DIA, low_di, ops, F32)


@gpu
@pytest.mark.parametrize("dtype,gate_dtype", [(F32, F32), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("rows,per,reverse", [(1000, 1, False), (1000, 1, True), (1000, 3, True), (50000, 1, False)])
def test_gates_whose_product_leaves_the_range(gs, dtype, gate_dtype, rows, per, reverse):
    """Gates of 2 and 1/2 over hundreds of rows: their products pass fp32's range (and over 50,000 rows
    that of 64 bits) while every state and gradient stays inside. Values are powers of 2, so also 16-bit
    gates hold them."""
    kinds, at = 6, 700
    x, gate = torch.zeros(rows, kinds), torch.ones(rows, kinds)
    dh, init, dfinal = torch.zeros(rows, kinds), torch.zeros(1, kinds), torch.zeros(1, kinds)
    gate[:, 0] = 2.0                                       # a zero state up to the last row
    x[-1, 0], dh[0, 0] = 3.0, 1.5                          # and a zero gradient down to the first
    gate[:, 1] = 2.0                                       # the same up to a reset
    gate[at, 1], x[at, 1], dh[at, 1] = 0.0, 1.0, 1.0
    gate[at + 1:, 1] = 0.5
    gate[at:at + 240, 2], init[0, 2] = 2.0, 2.0 ** -120    # a small state that grows
    gate[at:at + 200, 3], gate[at + 200:at + 290, 3] = 0.5, 2.0   # a large one that decays and grows again
    init[0, 3], dh[at + 100, 3] = 2.0 ** 60, 1.0
    gate[:at, 4], x[at, 4], dh[at, 4] = 2.0, 1.0, 2.0 ** -100     # a gradient between large gates
    gate[at - 150:at, 5], gate[at:at + 150, 5] = 2.0, 0.5  # up and down again
    init[0, 5], dfinal[0, 5] = 2.0 ** -60, 1.0
    gate[:at - 200, 4] = 1.0
    more = lambda t: t.repeat_interleave(per, 1)  # noqa: E731
    against(gs, more(x), gate, more(init), more(dh), more(dfinal), per, dtype, gate_dtype, reverse)


@gpu
@pytest.mark.parametrize("dtype,gate_dtype", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("channels,gates", [(1, 1), (3, 1), (40, 40), (40, 1), (40, 5), (21, 21), (35, 35), (301, 1), (1040, 2)])
def test_finite_inputs_give_finite_results(gs, dtype, gate_dtype, channels, gates):
    gen = torch.Generator(device=DEV).manual_seed(channels)
    for rows, sequences, offsets in ((700, 7, None), (4100, 1, None), (1283, 6, [0, 0, 700, 700, 701, 1280, 1280])):
        shape = (rows,) if offsets else (sequences, rows // sequences)
        leaves = [torch.randn(*shape, channels, generator=gen, device=DEV).to(dtype),
                  torch.rand(*shape, gates, generator=gen, device=DEV).to(gate_dtype),
                  torch.randn(sequences, channels, generator=gen, device=DEV)]
        leaves = [t.requires_grad_(True) for t in leaves]
        offs = None if offsets is None else torch.tensor(offsets, device=DEV)
        for reverse in (False, True):
            h, final = gs.gated_scan(*leaves, offsets=offs, reverse=reverse)
            grads = torch.autograd.grad((h, final), leaves, (torch.ones_like(h), torch.ones_like(final)))
            assert all(bool(torch.isfinite(t).all()) for t in (h, final) + grads)


@gpu
@pytest.mark.parametrize("rows", [3000, 60000])
def test_gates_that_grow_cost_little_more(gs, rows):
    """Products that leave the range take the chain's other form, not another order of magnitude."""
    x = torch.randn(rows, 64, device=DEV) * 1e-30
    times = []
    for high in (1.0, 1.02):
        g = torch.where(torch.rand(rows, 64, device=DEV) < 0.01, 0.0, high)
        for _ in range(3):
            h, _ = gs.gated_scan(x, g)
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        best = float("inf")
        for _ in range(10):
            start.record()
            gs.gated_scan(x, g)
            end.record()
            end.synchronize()
            best = min(best, start.elapsed_time(end))
        times.append(best)
        assert bool(torch.isfinite(h).all())
    assert times[1] < 4 * times[0] + 0.1, times


@gpu
@pytest.mark.parametrize("rows,lists", [(65536, 2048), (100, 7)])
@pytest.mark.parametrize("reverse", [False, True])
def test_a_long_run_of_empty_sequences(gs, rows, lists, reverse):
    """A million empty sequences between two others change no bit of what surrounds them, forward or
    backward, and in one run they take about the time that they take scattered."""
    gen = torch.Generator(device=DEV).manual_seed(rows)
    empty, channels = 1000000, 8
    cuts = torch.randint(0, rows + 1, (lists - 1,), generator=gen, device=DEV).sort().values
    bounds = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), rows)]).to(torch.int32)
    x = torch.randn(rows, channels, generator=gen, device=DEV)
    g = torch.rand(rows, 2, generator=gen, device=DEV)
    up = torch.randn(rows, channels, generator=gen, device=DEV)
    places = {"none": torch.zeros(lists, dtype=torch.int64, device=DEV)}
    places["run"] = places["none"].clone()
    places["run"][lists // 2] = empty
    places["scattered"] = torch.full_like(places["none"], empty // lists)
    out, times = {}, {}
    for kind, more in places.items():
        # before list s come more[s] empty ones
        offsets = torch.repeat_interleave(bounds, torch.cat([more + 1, more.new_ones(1)]))
        at = torch.arange(lists, device=DEV) + more.cumsum(0)     # the lists among all sequences
        init = torch.randn(offsets.shape[0] - 1, channels, generator=gen, device=DEV)
        init[at] = torch.arange(lists * channels, device=DEV).reshape(lists, channels).float() / channels
        dfinal = init.flip(1)
        leaves = [t.clone().requires_grad_(True) for t in (x, g, init)]

        def step():
            h, final = gs.gated_scan(leaves[0], leaves[1], initial=leaves[2], offsets=offsets, reverse=reverse)
            return (h, final) + torch.autograd.grad((h, final), leaves, (up, dfinal))

        h, final, dx, dg, dinit = step()
        none = torch.ones(init.shape[0], dtype=torch.bool, device=DEV)
        none[at] = False
        assert torch.equal(final[none], init[none]) and torch.equal(dinit[none], dfinal[none])
        out[kind] = (h, final[at], dx, dg, dinit[at])
        best = float("inf")
        for _ in range(5):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            step()
            end.record()
            end.synchronize()
            best = min(best, start.elapsed_time(end))
        times[kind] = best
    for kind in ("run", "scattered"):
        assert all(torch.equal(a, b) for a, b in zip(out["none"], out[kind])), kind
    assert times["run"] < 3 * times["scattered"] + 0.2, times


def test_forward_mode_derivatives_are_refused(gs):
    """A tangent would be lost without a word, as if the derivative were zero."""
    fw = torch.autograd.forward_ad
    x, g, init = torch.randn(4, 6), torch.rand(4, 6), torch.randn(1, 6)
    with fw.dual_level():
        duals = [fw.make_dual(t, torch.ones_like(t)) for t in (x, g, init)]
        for args in ((duals[0], g, init), (x, duals[1], init), (x, g, duals[2])):
            with pytest.raises(NotImplementedError):
                gs.gated_scan(*args)
    with pytest.raises(NotImplementedError):
        torch.func.jvp(lambda t: gs.gated_scan(t, g)[0], (x,), (x,))


@gpu
def test_forward_mode_levels_without_tangents(gs):
    fw = torch.autograd.forward_ad
    x, g = torch.randn(4, 6, device=DEV), torch.rand(4, 6, device=DEV)
    ref = gs.gated_scan(x, g)[0]
    with fw.dual_level():
        assert torch.equal(gs.gated_scan(x, g)[0], ref)
        for wanted in (False, True):
            leaf = x.clone().requires_grad_(wanted)
            with pytest.raises(NotImplementedError):
                gs.gated_scan(fw.make_dual(leaf, torch.ones_like(x)), g)


@gpu
def test_offsets_are_looked_at_without_rows(gs):
    nat = importlib.import_module("3dgs_from_scratch_b200._native")
    init = torch.randn(2, 6, device=DEV, requires_grad=True)
    for kind, layout in ((F32, torch.zeros(0, 6, device=DEV)), (F32, torch.zeros(9, 12, device=DEV)[9:, 3:9])):
        x = layout.to(kind)
        for offsets, error in (([0, 0, 0], nat.GS_OK), ([0, 0, 5], nat.GS_ERR_INVALID_ARGUMENT),
                               ([0, -1, 0], nat.GS_ERR_INVALID_ARGUMENT)):
            assert nat.query("gs_check_status", nat.stream_ptr()) == nat.GS_OK
            offs = torch.tensor(offsets, device=DEV)
            h, final = gs.gated_scan(x, x, initial=init, offsets=offs)
            assert nat.query("gs_check_status", nat.stream_ptr()) == error
            assert h.shape == (0, 6)
            if error == nat.GS_OK:
                assert torch.equal(final, init)
                (dinit,) = torch.autograd.grad(final.square().sum(), init)
                assert torch.equal(dinit, 2 * init.detach())
                assert float(gs.gated_scan(x, x, offsets=offs)[1].abs().max()) == 0.0
