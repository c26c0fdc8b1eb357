"""The multi-tensor AdamW step (32-bit and 8-bit states), the global gradient norm and the decoding of
8-bit moments on the GPU, against a 64-bit oracle."""
import math

import pytest
import torch

from . import adamw_oracle as orc

pytestmark = pytest.mark.gpu
DEV = "cuda"
HYPER = dict(lr=1e-2, beta_1=0.9, beta_2=0.999, epsilon=1e-7, weight_decay=0.1)


def rand(*shape, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g) * scale


def make(sizes, layout, grad_dtype=torch.float32, seed=0):
    """(params, grads, buffers): tensors of their own, views at multiples of 64, or views at odd places;
    the buffers' other places hold 7."""
    ps, gs = [], []
    for i, n in enumerate(sizes):
        ps.append(rand(n, seed=seed + 2 * i, scale=0.5))
        gs.append(rand(n, seed=seed + 2 * i + 1, scale=10.0 ** (i % 5 - 3)).to(grad_dtype))
    if layout == "own":
        return [p.to(DEV) for p in ps], [g.to(DEV) for g in gs], None
    gap = {"arena": 0, "odd": 1, "half": 4}[layout]  # "half": multiples of 8 bytes (bf16), or of 16
    offs, total = [], gap
    for n in sizes:
        offs.append(total)
        total += orc.pad64(n) + gap
    wb = torch.full((total + 64,), 7.0, device=DEV)
    gb = torch.full((total + 64,), 7.0, device=DEV, dtype=grad_dtype)
    pv, gv = [wb[o:o + n] for o, n in zip(offs, sizes)], [gb[o:o + n] for o, n in zip(offs, sizes)]
    for v, t in zip(pv + gv, ps + gs):
        v.copy_(t)
    inside = torch.zeros(total + 64, dtype=torch.bool, device=DEV)
    for o, n in zip(offs, sizes):
        inside[o:o + n] = True
    return pv, gv, (wb, gb, ~inside)


def moments_for(grads, bits, seed):
    """Flat fp32 (m, v) of a state in mid-training; padding is zero."""
    g, offs = orc.place(grads)
    r = torch.Generator().manual_seed(seed)
    size = g.abs() + 1e-6 * (g != 0)
    m = torch.randn(g.shape, generator=r, dtype=torch.float64) * size * 0.3
    v = size ** 2 * (torch.rand(g.shape, generator=r, dtype=torch.float64) * 2 + 0.01)
    return m.float(), v.float()


def start(params, grads, bits, t0, decay, seed=5):
    from idc_models_amd.ops import optim
    table = optim.TensorTable(grads, params, decay=decay)
    st = optim.AdamWState(table, bits=bits)
    m, v = moments_for(grads, bits, seed)
    if t0:
        st.load_moments(m, v)
        st.set_step(t0)
    return table, st


def state_values(st):
    """(m, v) in fp64 on the CPU, by the oracle's own decoding."""
    if st.bits == 32:
        return st.m.double().cpu(), st.v.double().cpu()
    sc = st.scales.cpu()
    r = orc.code_values(st.v.cpu(), sc[:, 1], orc.ROOT_BITS)
    return orc.code_values(st.m.cpu(), sc[:, 0], orc.M_BITS), r * r


def check_step(params, grads, table, st, decay, grad_scale=1.0, clip=0.0, hyper=HYPER, call=None):
    """Runs one step and compares everything with the oracle."""
    from idc_models_amd.ops import optim
    w0, offs = orc.place(params)
    g0, _ = orc.place(grads)
    mask = torch.zeros_like(w0)
    for o, p, d in zip(offs, params, decay):
        mask[o:o + p.numel()] = float(d)
    m0, v0 = state_values(st)
    t = int(st.step[0]) + 1
    total = orc.norm(grads)
    if call is None:
        optim.adamw_(table, st, hyper["lr"], hyper["beta_1"], hyper["beta_2"], hyper["epsilon"],
                     hyper["weight_decay"], grad_scale, clip_norm=clip)
    else:
        call()
    torch.cuda.synchronize()
    w1, m1, v1, root, tw, tm, tv, tr = orc.step(
        w0, g0, m0, v0, t, hyper["lr"], hyper["beta_1"], hyper["beta_2"], hyper["epsilon"], hyper["weight_decay"],
        mask, grad_scale, clip, total)
    got, _ = orc.place(params)
    orc.within(got, w1, tw)
    assert bool((st.step == t).all())
    if clip:
        assert float(st.norm) == pytest.approx(total, rel=2 * orc.U) or not math.isfinite(total)
    m, v = state_values(st)
    if st.bits == 32 or not m.numel():
        orc.within(m, m1, tm)
        orc.within(v, v1, tv)
        return
    low, high = orc.hash_bits(m1.numel(), t)
    for have, x, bits, mantissa, slack in ((m, m1, low, orc.M_BITS, 32 * orc.U), (v.sqrt(), root, high, orc.ROOT_BITS, 16 * orc.U)):
        # where b1*m and (1-b1)*g cancel, m's relative error is larger: its own bound
        if mantissa == orc.M_BITS:
            slack = torch.where(x == 0, torch.full_like(x, slack), torch.maximum(torch.full_like(x, slack), tm / x.abs().clamp(min=1e-300))).clamp(max=0.5)
            lo, hi, open_ = bounds_each(x, mantissa, bits, slack)
        else:
            lo, hi, open_ = orc.code_bounds(x, mantissa, bits, slack)
            # a second moment below fp32's smallest normal number may be cut to zero
            open_ = open_ | (x.view(-1, orc.BLOCK).amax(1) < 2.0 ** -62).repeat_interleave(orc.BLOCK)
        same = (have == lo) | (have == hi) | (torch.isnan(have) & torch.isnan(lo))
        assert bool((same | open_).all()), int((~(same | open_)).sum())
        assert float((lo != hi).double().mean()) < 0.01 or have.numel() < 2000


def bounds_each(x, mantissa, r16, slack):
    """code_bounds with a slack for each element: the oracle's cut of both ends; the block's scale is
    taken from x itself."""
    block_slack = float(slack.view(-1, orc.BLOCK).gather(1, x.abs().nan_to_num(0, 0, 0).view(-1, orc.BLOCK).argmax(1)[:, None]).max())
    lo, hi, open_ = orc.code_bounds(x, mantissa, r16, 1e-9)
    one = 1 << mantissa
    a = x.abs().view(-1, orc.BLOCK)
    bad = ~torch.isfinite(a).all(1)
    a = torch.where(bad[:, None], torch.zeros_like(a), a)
    k = torch.log2(torch.clamp(a.amax(1), min=2.0 ** -149) / ((2 * one - 1) * 2.0 ** 14))
    open_ = open_ | ((k - k.round()).abs() < 4 * block_slack).repeat_interleave(orc.BLOCK)
    unit = (2.0 ** torch.clamp(torch.ceil(k), min=-126.0)).repeat_interleave(orc.BLOCK)
    ends = []
    for f in (1 - slack, 1 + slack):
        y = a.view(-1) * f / unit
        q = 2.0 ** torch.clamp(torch.floor(torch.log2(torch.clamp(y, min=1.0))) - mantissa, min=0.0)
        c = torch.floor(y / q + (r16.double() + 0.5) / 65536.0) * q * unit
        c = torch.where(x < 0, -c, c)
        c[bad.repeat_interleave(orc.BLOCK)] = math.nan
        ends.append(c)
    return ends[0], ends[1], open_


SIZES = [[1], [3, 64, 65, 1], [2048], [2047, 0, 2049, 5], [4096 + 17, 63, 128], [1] * 70, [30011, 1025], [0, 0]]


@pytest.mark.parametrize("layout", ["own", "arena", "odd", "half"])
@pytest.mark.parametrize("grad_dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("bits", [32, 8])
def test_step_matches_the_formula(bits, grad_dtype, layout):
    for k, sizes in enumerate(SIZES):
        for t0, clip, gs in ((0, 0.0, 1.0), (37, 0.5, -0.25)):
            print(bits, grad_dtype, layout, sizes[:4], t0, flush=True)
            params, grads, buf = make(sizes, layout, grad_dtype, seed=100 * k)
            decay = [i % 2 == 0 for i in range(len(sizes))]
            table, st = start(params, grads, bits, t0, decay)
            for _ in range(2):  # the second step starts from a state that the kernel wrote
                check_step(params, grads, table, st, decay, gs, clip)
            if buf is not None:  # what lies between the tensors stays
                wb, gb, outside = buf
                assert bool((wb[outside] == 7.0).all()) and bool((gb[outside] == 7.0).all())


def test_more_pieces_than_workgroups():
    """More pieces than workgroups; the larger pieces of large tables; beyond the caches."""
    for sizes, bits in (([2048 * 700 + 3, 2048 * 900, 77], 32), ([2048 * 700 + 3, 2048 * 900, 77], 8),
                        ([4096 * 700 + 3, 4096 * 400, 77], 32), ([4096 * 700 + 3, 4096 * 400, 77], 8),
                        ([4096 * 2800 + 3, 77], 8)):
        params, grads, _ = make(sizes, "own", seed=9)
        decay = [i != 1 for i in range(len(sizes))]
        table, st = start(params, grads, bits, 5, decay)
        assert table.nchunks > 1024 and table.chunk == (2048 if sizes[0] < 4096 * 700 else 4096)
        check_step(params, grads, table, st, decay, 1.0, 1.0)


@pytest.mark.parametrize("grad_dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("bits", [32, 8])
def test_the_largest_tables(bits, grad_dtype):
    """A workgroup for each piece, and a launch that counts: two clipped steps; the ends of both
    tensors against the oracle."""
    from idc_models_amd.ops import optim
    n = [8192 * 4096 + 4096 + 5, 777]
    gen = torch.Generator(device=DEV).manual_seed(3)
    params = [torch.randn(k, device=DEV, generator=gen) for k in n]
    grads = [torch.randn(k, device=DEV, generator=gen).to(grad_dtype) for k in n]
    table = optim.TensorTable(grads, params, decay=[True, False])
    st = optim.AdamWState(table, bits=bits)
    assert table.nchunks >= 8192
    word = torch.ones(1, dtype=torch.int32, device=DEV)
    before = params[1].clone()
    optim.adamw_(table, st, **HYPER, skip=word, clip_norm=10.0)
    assert int(st.step[0]) == 0 and torch.equal(before, params[1]) and int(st.m.view(torch.uint8).max()) == 0
    total = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    first = (n[0] - 10000) // 64 * 64
    parts = [(0, 0, 0, 8192), (0, first, first, n[0]), (1, 0, table.offsets[1], 777)]  # tensor, from, place, to
    for t in (1, 2):
        olds = [(params[i][a:b].double().cpu(), grads[i][a:b].double().cpu()) for i, a, _, b in parts]
        states = [slice_values(st, at, orc.pad64(b - a)) for _, a, at, b in parts]
        optim.adamw_(table, st, **HYPER, clip_norm=10.0)
        assert float(st.norm) == pytest.approx(total, rel=2 * orc.U) and bool((st.step == t).all())
        for (i, a, at, b), (w0, g), (m0, r0) in zip(parts, olds, states):
            k, pad = b - a, orc.pad64(b - a)
            ext = lambda x: torch.cat([x, torch.zeros(pad - k, dtype=torch.float64)])
            w1, m1, v1, root, tw, tm, tv, tr = orc.step(ext(w0), ext(g), m0, r0 * r0, t, HYPER["lr"], 0.9, 0.999, 1e-7, 0.1,
                                                        torch.full((pad,), float(i == 0), dtype=torch.float64), 1.0, 10.0, total)
            orc.within(params[i][a:b], w1[:k], tw[:k])
            m, r = slice_values(st, at, pad)
            if bits == 32:
                orc.within(m, m1, tm)
                orc.within(r, root, tr + orc.U * root)
                continue
            low, high = orc.hash_bits(pad, t, start=at)
            slack = torch.where(m1 == 0, torch.zeros_like(m1), tm / m1.abs().clamp(min=1e-300)).clamp(min=32 * orc.U, max=0.5)
            for have, (lo, hi, open_) in ((m, bounds_each(m1, 3, low, slack)), (r, orc.code_bounds(root, 4, high, 16 * orc.U))):
                assert bool(((have == lo) | (have == hi) | open_).all())


def slice_values(st, at, n):
    """First moments and roots (fp64) of n places of the state from a multiple of 64 on."""
    if st.bits == 32:
        return st.m[at:at + n].double().cpu(), st.v[at:at + n].double().sqrt().cpu()
    sc = st.scales[at // 64:(at + n) // 64].cpu()
    return (orc.code_values(st.m[at:at + n].cpu(), sc[:, 0], 3), orc.code_values(st.v[at:at + n].cpu(), sc[:, 1], 4))


@pytest.mark.parametrize("bits", [32, 8])
def test_other_betas_and_late_steps(bits):
    for b1, b2, t0 in ((0.0, 0.0, 0), (0.0, 0.99, 3), (0.95, 0.0, 1), (0.9, 0.9999, 10 ** 6), (0.99, 0.999, 1)):
        params, grads, _ = make([1000, 65], "own", seed=3)
        table, st = start(params, grads, bits, t0, [True, True])
        check_step(params, grads, table, st, [True, True], hyper=dict(HYPER, beta_1=b1, beta_2=b2, epsilon=1e-8))


def test_axes_in_another_order():
    """Weights and gradients that are dense but not contiguous: the order in memory counts."""
    from idc_models_amd.ops import optim
    p = rand(3, 5, 7, 9, seed=1).to(DEV).permute(3, 0, 2, 1)
    g = rand(3, 5, 7, 9, seed=2).to(DEV).permute(3, 0, 2, 1)
    p2, g2 = p.clone(), g.clone()  # same order again
    table, st = start([p], [g], 32, 0, [True])
    check_step([p], [g], table, st, [True])
    c, d = p2.contiguous(), g2.contiguous()
    t2 = optim.TensorTable([d], [c])
    s2 = optim.AdamWState(t2)
    optim.adamw_(t2, s2, **HYPER)
    assert torch.equal(c, p)
    assert t2.split(s2.m)[0].shape == c.shape and torch.equal(t2.split(s2.m)[0], st.m[:p.numel()].as_strided(p.shape, p.stride()))


@pytest.mark.parametrize("bits", [32, 8])
def test_values_at_the_ends_of_the_range(bits):
    """Zeros, the smallest and the largest squares, signs; no gradient may disturb another block."""
    n = 64 * 8
    g = torch.zeros(n)
    g[64:128] = 1e-22          # squares vanish in fp32: moves by its first moment alone
    g[128:192] = torch.linspace(-1, 1, 64) * 1e-12
    g[192:256] = 1e18
    g[256] = 3.0               # alone in its block
    g[320:384] = torch.tensor([2.0 ** -k for k in range(64)])
    g[384:448] = -g[320:384]
    g[448:512] = -0.0
    p, g = rand(n, seed=4).to(DEV), g.to(DEV)
    hyper = dict(HYPER, epsilon=1e-3)  # 1e-22 squared is no fp32 number: the quotient is m / eps there
    table, st = start([p], [g], bits, 0, [True])
    for _ in range(3):
        check_step([p], [g], table, st, [True], hyper=hyper)
    assert bool((st.m[448:] % 128 == 0).all()) if bits == 8 else bool((st.m[448:] == 0).all())


def test_values_that_are_not_finite():
    """fp32 states: as the formula.  8-bit states: the block of 64 turns to NaN, and no other."""
    from idc_models_amd.ops import optim
    for bits in (32, 8):
        for bad in (math.nan, math.inf, -math.inf):
            p, g = rand(300, seed=4).to(DEV), rand(300, seed=5).to(DEV)
            g[70] = bad
            table, st = start([p], [g], bits, 3, [True])
            check_step([p], [g], table, st, [True])
            m, v = state_values(st)
            hit = torch.isnan(m) | torch.isinf(m)
            assert hit.nonzero().flatten().tolist() == ([70] if bits == 32 else list(range(64, 128)))
            g[70] = 1.0
            check_step([p], [g], table, st, [True])
            keep = torch.ones(300, dtype=torch.bool)
            keep[64:128] = False
            assert bool(torch.isfinite(p.cpu()[keep]).all())
            if bits == 8:
                assert bool(torch.isnan(p[64:128]).all()) and bool((st.scales[1] == 255).all())
                assert bool(torch.isnan(st.decode()[0][64:128]).all())
            # a clipped step: the norm is not finite, every gradient becomes NaN
            g[70] = bad
            optim.adamw_(table, st, **HYPER, clip_norm=1.0)
            assert bool(torch.isnan(p).all()) and not math.isfinite(float(st.norm))


@pytest.mark.parametrize("bits", [32, 8])
def test_second_moment_that_leaves_fp32(bits):
    """A square beyond fp32: the first moment stays finite, the weight keeps still in this step; an 8-bit
    block reads as NaN from then on, by its second moment alone."""
    p, g = rand(200, seed=4).to(DEV), rand(200, seed=5).to(DEV)
    table, st = start([p], [g], bits, 3, [True])
    assert bool(torch.isfinite(state_values(st)[1]).all())
    g[70] = 1e25
    check_step_fp32(p, g, table, st)
    m, v = state_values(st)
    assert bool(torch.isfinite(m).all()) and bool(torch.isfinite(p).all())
    bad = (~torch.isfinite(v)).nonzero().flatten().tolist()
    assert bad == ([70] if bits == 32 else list(range(64, 128)))


def check_step_fp32(p, g, table, st):
    """One step where the oracle's second moment has to leave fp32's range as fp32 does."""
    from idc_models_amd.ops import optim
    w0, _ = orc.place([p])
    m0, v0 = state_values(st)
    g0, _ = orc.place([g])
    optim.adamw_(table, st, **HYPER)
    g1 = torch.where(g0 > 1e20, torch.full_like(g0, 1e200), g0)
    w1, *_, tw, _, _, _ = orc.step(w0, g1, m0, v0, int(st.step[0]), HYPER["lr"], 0.9, 0.999, 1e-7, 0.1, torch.ones_like(w0))
    keep = g0 < 1e20
    got, _ = orc.place([p])
    orc.within(got[keep], w1[keep], tw[keep])
    i = int((~keep).nonzero()[0])  # m / inf: only the decay is left
    assert float(got[i]) == pytest.approx(float(w0[i]) * (1 - HYPER["lr"] * HYPER["weight_decay"]), rel=1e-6)


def test_refused_calls():
    from idc_models_amd.ops import optim
    p, g = torch.zeros(100, device=DEV), torch.zeros(100, device=DEV)
    table = optim.TensorTable([g], [p])
    st = optim.AdamWState(table)
    other = optim.AdamWState(optim.TensorTable([g.new_zeros(200)], [p.new_zeros(200)]))
    norm_only = optim.TensorTable([g])
    for call in (lambda: optim.adamw_(table, other, 1e-3), lambda: optim.adamw_(norm_only, st, 1e-3),
                 lambda: optim.AdamWState(norm_only), lambda: optim.AdamWState(table, bits=4), lambda: st.decode(),
                 lambda: optim.adamw_(table, st, math.nan), lambda: optim.adamw_(table, st, 1e-3, grad_scale=math.inf),
                 lambda: optim.adamw_(table, st, 1e-3, skip=torch.zeros(1, device=DEV)),
                 lambda: optim.adamw_(table, st, 1e-3, skip=torch.zeros(1, dtype=torch.int32)),
                 lambda: optim.AdamWState(table, bits=8).decode(torch.float16),
                 lambda: st.load_moments(st.m[:64], st.v)):
        with pytest.raises(ValueError):
            call()
    assert int(st.step[0]) == 0


def test_scale_borders_are_exact():
    """A block whose largest value is exactly a unit's largest code keeps that unit; the next number up
    takes the next one."""
    from idc_models_amd.ops import optim
    for top, up in ((15.0 * 2 ** 14, 1), (31.0 * 2 ** 14, 1)):
        p, g = torch.zeros(128, device=DEV), torch.zeros(128, device=DEV)
        first = top == 15.0 * 2 ** 14
        g[0], g[64] = top, float(torch.nextafter(torch.tensor(top), torch.tensor(1e30)))
        table = optim.TensorTable([g], [p])
        st = optim.AdamWState(table, bits=8)
        optim.adamw_(table, st, 0.0, 0.0, 0.0, 1e-7, 0.0)  # m = g, v = g^2
        s = st.scales.cpu()[:, 0 if first else 1]
        if first:
            assert s.tolist() == [127, 128]
            assert st.m.cpu()[0] == 127
            m, _ = st.decode()
            assert float(m[0]) == top
        else:
            assert int(s[0]) == 127 and float(st.decode()[1][0]) == top


@pytest.mark.parametrize("bits", [32, 8])
def test_skip_word(bits):
    from idc_models_amd.ops import optim
    p, g = rand(3000, seed=4).to(DEV), rand(3000, seed=5).to(DEV)
    table, st = start([p], [g], bits, 3, [True])
    before = [p.clone()] + [t.clone() for t in st.tensors().values()]
    word = torch.ones(1, dtype=torch.int32, device=DEV)
    optim.adamw_(table, st, **HYPER, skip=word)
    assert all(torch.equal(a, b) for a, b in zip(before, [p] + list(st.tensors().values())))
    word.zero_()
    check_step([p], [g], table, st, [True], call=lambda: optim.adamw_(table, st, **HYPER, skip=word))


@pytest.mark.parametrize("bits", [32, 8])
def test_graph_replays_count_steps(bits):
    """A captured clipped step, replayed with eager work in between, gives the eager steps' bits."""
    from idc_models_amd.ops import optim
    sizes = [5000, 64, 3]
    pa, ga, _ = make(sizes, "own", seed=1)
    pb, gb = [t.clone() for t in pa], [t.clone() for t in ga]
    ta, sa = start(pa, ga, bits, 0, [True] * 3)
    tb, sb = start(pb, gb, bits, 0, [True] * 3)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        optim.adamw_(tb, sb, **HYPER, clip_norm=0.3)
        total = optim.global_norm(tb)
    for k in range(5):
        for a, b in zip(ga, gb):
            a.mul_(1.5).add_(0.01 * k)
            b.copy_(a)
        optim.adamw_(ta, sa, **HYPER, clip_norm=0.3)
        graph.replay()
        eager = optim.global_norm(ta)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(pa, pb))
        assert all(torch.equal(a, b) for a, b in zip(sa.tensors().values(), sb.tensors().values()))
        assert torch.equal(total, eager) and int(sb.step[7]) == k + 1


def test_same_bits_every_time_and_on_another_stream():
    from idc_models_amd.ops import optim
    for bits in (32, 8):
        runs = []
        for other in (False, True):
            params, grads, _ = make([70001, 3, 5000], "own", seed=2)
            table, st = start(params, grads, bits, 3, [True, False, True])
            torch.cuda.synchronize()
            s = torch.cuda.Stream() if other else torch.cuda.current_stream()
            with torch.cuda.stream(s):
                for _ in range(3):
                    optim.adamw_(table, st, **HYPER, clip_norm=0.7)
                n = optim.global_norm(table)
            s.synchronize()
            runs.append([n] + params + list(st.tensors().values()))
        assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("grad_dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_global_norm(grad_dtype):
    from idc_models_amd.ops.optim import TensorTable, global_norm
    for sizes in ([1], [0], [3, 64, 0, 65], [2048 * 8], [2048 * 32 - 3], [2048 * 32 + 1], [5] * 32, [77] * 33, [2048 * 1500 + 5, 9, 1]):
        for layout in ("own", "odd", "half"):
            _, grads, _ = make(sizes, layout, grad_dtype, seed=7)
            want = orc.norm(grads)
            got = global_norm(TensorTable(grads))
            assert got.shape == () and got.dtype == torch.float32
            # squares and sums in fp64, one rounding to fp32
            assert abs(float(got) - want) <= 2 * orc.U * want
    for value in (1e-30, 1e30, math.inf, math.nan):  # squares beyond fp32, and what is not finite
        g = torch.full((5000,), value, device=DEV, dtype=grad_dtype)
        got, want = float(global_norm(TensorTable([g, g]))), math.sqrt(10000) * float(g[0])  # one tensor twice: counts twice
        assert got == pytest.approx(want, rel=1e-6, nan_ok=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_decode_gives_every_code(dtype):
    from idc_models_amd.ops import optim
    p = torch.zeros(256 * 64 + 1, device=DEV)
    st = optim.AdamWState(optim.TensorTable([p.clone()], [p]), bits=8)
    n = st.numel
    codes = torch.arange(n, device=DEV)
    st.m.copy_((codes % 256).to(torch.uint8))
    st.v.copy_((codes // 7 % 256).to(torch.uint8))
    # units from 2^-126 to 2^100: every value is a normal number below fp32's (and bf16's) largest
    st.scales.copy_(torch.stack([1 + torch.arange(n // 64, device=DEV) % 227, 227 - torch.arange(n // 64, device=DEV) % 227], 1).to(torch.uint8))
    st.scales[3] = 255
    st.scales[5] = 0
    st.m[5 * 64:6 * 64] = 0
    st.v[5 * 64:6 * 64] = 0
    m, r = st.decode(dtype)
    assert m.dtype == dtype and r.dtype == dtype
    sc = st.scales.cpu()
    for got, codes, col, bits in ((m, st.m, 0, orc.M_BITS), (r, st.v, 1, orc.ROOT_BITS)):
        want = orc.code_values(codes.cpu(), sc[:, col], bits)
        assert torch.equal(got.double().cpu().nan_to_num(-5.0), want.nan_to_num(-5.0))


def test_places_beyond_32_bits():
    """A state longer than 2^32: the last tensor's weights, codes and dither are those of its place."""
    from idc_models_amd.ops import optim
    free, _ = torch.cuda.mem_get_info()
    if free < 60e9:
        pytest.skip("needs 60 GB of free GPU memory")
    big = (1 << 32) + 4096
    p0 = torch.zeros(big, device=DEV)
    g0 = torch.zeros(big, device=DEV, dtype=torch.bfloat16)
    g0[-1] = 1.0
    p1, g1 = rand(777, seed=1).to(DEV), rand(777, seed=2).to(DEV).bfloat16()
    table = optim.TensorTable([g0, g1], [p0, p1])
    st = optim.AdamWState(table, bits=8)
    w0, g = p1.double().cpu(), g1.double().cpu()
    z = torch.zeros_like(w0)
    for t in (1,):
        optim.adamw_(table, st, **HYPER)
    w1, m1, v1, root, tw, *_ = orc.step(w0, g, z, z, 1, HYPER["lr"], 0.9, 0.999, 1e-7, 0.1, torch.ones_like(w0))
    orc.within(p1, w1, tw)
    low, high = orc.hash_bits(orc.pad64(777), 1, start=table.offsets[1])
    pad = torch.zeros(orc.pad64(777) - 777, dtype=torch.float64)
    sc = st.scales[table.offsets[1] // 64:].cpu()
    for codes, col, x, bits, mantissa in ((st.m, 0, m1, low, 3), (st.v, 1, root, high, 4)):
        have = orc.code_values(codes[table.offsets[1]:].cpu(), sc[:, col], mantissa)
        lo, hi, open_ = orc.code_bounds(torch.cat([x, pad]), mantissa, bits, 32 * orc.U)
        assert bool(((have == lo) | (have == hi) | open_).all())
    # the big tensor: its last element moved by lr, the others hold zeros
    assert float(p0[-1]) == pytest.approx(-HYPER["lr"], rel=1e-5) and float(p0[:-1].abs().max()) == 0.0
    n = optim.global_norm(table)
    assert float(n) == pytest.approx(math.sqrt(1.0 + float(g.square().sum())), rel=1e-6)


@pytest.mark.parametrize("bits", [32, 8])
def test_weights_whose_storage_is_replaced(bits):
    """A table over Parameters that an arena (or p.data = x) moves elsewhere: the step is refused and
    changes nothing, neither the weights nor memory that other tensors have got since."""
    from idc_models_amd.engine import ParamArena
    from idc_models_amd.ops import optim
    ps = [torch.nn.Parameter(rand(5000, seed=i).to(DEV)) for i in range(3)]
    gs = [rand(5000, seed=10 + i).to(DEV) for i in range(3)]
    table = optim.TensorTable(gs, ps)
    st = optim.AdamWState(table, bits=bits)
    optim.adamw_(table, st, **HYPER)  # in place: fine
    table.check()
    arena = ParamArena(ps)
    before = [p.detach().clone() for p in ps]
    others = [torch.full((5000,), 7.0, device=DEV) for _ in range(50)]
    for _ in range(2):
        with pytest.raises(ValueError, match="other storage"):
            optim.adamw_(table, st, **HYPER)
    with pytest.raises(ValueError, match="other storage"):
        table.check()
    torch.cuda.synchronize()
    assert int(st.step[0]) == 1 and all(torch.equal(p, b) for p, b in zip(ps, before))
    assert all(bool((o == 7.0).all()) for o in others)
    table = optim.TensorTable([arena.grad_of(p) for p in ps], ps)  # a new table takes them where they are
    optim.adamw_(table, st, **HYPER)
    assert int(st.step[0]) == 2
    # tensors that autograd does not know: the memory stays the table's own, check() sees the change
    w, g = rand(3000, seed=1).to(DEV), rand(3000, seed=2).to(DEV)
    table = optim.TensorTable([g], [w])
    st = optim.AdamWState(table, bits=bits)
    g.data = torch.zeros(3000, device=DEV)
    with pytest.raises(ValueError, match="other storage"):
        table.check()
    w.data = torch.zeros(3000, device=DEV)
    others = [torch.full((3000,), 7.0, device=DEV) for _ in range(50)]
    optim.adamw_(table, st, **HYPER)
    torch.cuda.synchronize()
    assert all(bool((o == 7.0).all()) for o in others) and float(w.abs().max()) == 0.0


def test_state_and_tables_of_the_same_length():
    """A state goes with its tensors' sizes: tables in another order are refused, a second table of the same tensors
    is fine."""
    from idc_models_amd.ops import optim
    ps, gs = [rand(n, seed=n).to(DEV) for n in (100, 30)], [rand(n, seed=n + 1).to(DEV) for n in (100, 30)]
    st = optim.AdamWState(optim.TensorTable(gs, ps))
    before = [p.clone() for p in ps]
    with pytest.raises(ValueError, match="another table"):
        optim.adamw_(optim.TensorTable(gs[::-1], ps[::-1]), st, **HYPER)
    assert int(st.step[0]) == 0 and all(torch.equal(p, b) for p, b in zip(ps, before))
    gs = [g.clone() for g in gs]
    check_step(ps, gs, optim.TensorTable(gs, ps), st, [True, True])


def test_a_second_backward_after_a_step_raises():
    """As after torch's own optimizers: the graph saved the weights that the step has changed.  A refused
    call changes nothing, so the graph stays good."""
    from idc_models_amd.ops import optim
    lin = torch.nn.Linear(70, 33).to(DEV)
    x = rand(8, 70, seed=1).to(DEV).requires_grad_()
    lin(x).square().sum().backward()
    table = optim.TensorTable([p.grad for p in lin.parameters()], list(lin.parameters()))
    st = optim.AdamWState(table)
    y = lin(x).square().sum()
    y.backward(retain_graph=True)
    with pytest.raises(ValueError):
        optim.adamw_(table, st, -1.0)
    y.backward(retain_graph=True)
    optim.adamw_(table, st, **HYPER)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    for _ in range(2):  # steps whose graphs are new go on
        for p in lin.parameters():
            p.grad.zero_()
        lin(x).square().sum().backward()
        check_step([p for p in lin.parameters()], [p.grad for p in lin.parameters()], table, st, [True, True])


def test_version_of_captured_steps():
    """A step over Parameters can be captured; each eager call is one change for autograd."""
    from idc_models_amd.ops import optim
    p = torch.nn.Parameter(rand(500, seed=1).to(DEV))
    g = rand(500, seed=2).to(DEV)
    table = optim.TensorTable([g], [p])
    st = optim.AdamWState(table)
    v = p._version
    optim.adamw_(table, st, **HYPER)
    assert p._version > v
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        optim.adamw_(table, st, **HYPER)
    for _ in range(3):
        check_step([p], [g], table, st, [True], call=graph.replay)


LARGE = {"2048-element pieces": ([2048 * 700 + 3, 2048 * 900, 77], 2048), "4096-element pieces": ([4096 * 700 + 3, 4096 * 400, 77], 4096),
         "past the caches": ([4096 * 2800 + 3, 77], 4096)}  # (32 bits: from 1,366 pieces on; 8 bits: from 2,731)


@pytest.mark.parametrize("sizes", LARGE, ids=lambda k: k.replace(" ", "-"))
@pytest.mark.parametrize("grad_dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("bits", [32, 8])
def test_every_kind_of_large_table(bits, grad_dtype, sizes):
    """More pieces than workgroups: both piece sizes, cached and past the caches, either width and gradient type;
    tensors of their own, and at addresses that vector accesses cannot use."""
    sizes, chunk = LARGE[sizes]
    for layout in ("own", "odd"):
        params, grads, buf = make(sizes, layout, grad_dtype, seed=9)
        decay = [i != 1 for i in range(len(sizes))]
        table, st = start(params, grads, bits, 5, decay)
        assert 1024 < table.nchunks < 8192 and table.chunk == chunk
        assert (table.nchunks * chunk * (12 if bits == 8 else 24) >= 128 << 20) == (len(sizes) == 2)
        check_step(params, grads, table, st, decay, 1.0, 1.0)
        if buf is not None:
            wb, gb, outside = buf
            assert bool((wb[outside] == 7.0).all()) and bool((gb[outside] == 7.0).all())


@pytest.mark.parametrize("grad_dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_global_norm_of_large_pieces(grad_dtype):
    """Tables of 4096-element pieces; pieces of zeros and of values whose squares are no fp32 numbers among them."""
    from idc_models_amd.ops.optim import TensorTable, global_norm
    n = 4096 * 1100 + 2048 + 5  # its last pieces have 4096 and 2053 elements
    for layout in ("own", "odd"):
        _, grads, _ = make([n, 2048, 9], layout, grad_dtype, seed=7)
        table = TensorTable(grads)
        assert table.chunk == 4096 and table.nchunks == 1103
        for value in (None, 0.0, 1e-30, 1e25):
            if value is not None:
                grads[0][:4096 * 8].view(8, 4096)[::2] = value
            want = orc.norm(grads)
            # one rounding to fp32; bf16: sums of 16 exact squares in fp32, 4 roundings deep, which the root halves
            tol = orc.U if grad_dtype is torch.float32 else 3 * orc.U
            assert abs(float(global_norm(table)) - want) <= (tol + 2.0 ** -40) * want
