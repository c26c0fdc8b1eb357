"""AdamW in the fused program, the eager backend, client-batched federated training and checkpoints on
the GPU."""
import copy
import math

import pytest
import torch

from . import adamw_oracle as orc

pytestmark = pytest.mark.gpu
DEV = "cuda"


def model(opt, arch="densenet121", backend="fused", seed=0, **kw):
    from idc_models_amd.engine import Model
    from idc_models_amd.models import build_model
    m = Model(build_model(arch, None, num_outputs=1, seed=seed), device=DEV)
    m.compile(opt, "binary_crossentropy", [], backend=backend, **kw)
    return m


def batch(n=8, seed=1):
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(0, 256, (n, 50, 50, 3), generator=g, dtype=torch.uint8).to(DEV),
            torch.randint(0, 2, (n,), generator=g).to(DEV))


def values(opt):
    if opt.state_bits == 32:
        return opt.m.double().cpu(), opt.v.double().cpu()
    sc = opt.scales.cpu()
    return orc.code_values(opt.m.cpu(), sc[:, 0], 3), orc.code_values(opt.v.cpu(), sc[:, 1], 4) ** 2


def mask_of(m, decay):
    out = torch.zeros(m.arena.numel, dtype=torch.float64)
    for p, s in zip(m.arena.params, m.arena.slots):
        out[s.offset:s.offset + s.numel] = float(decay == "all" or p.dim() > 1)
    return out


@pytest.mark.parametrize("arch,bits,clip,decay", [("densenet121", 32, 0.1, "kernels"), ("densenet121", 8, None, "all"),
                                                  ("mobilenetv2", 8, 0.1, "kernels"), ("vgg16", 32, None, "all")])
def test_fused_steps_match_the_formula(arch, bits, clip, decay):
    """Training steps of the fused program (the update is part of a replayed graph): the weights after
    each step follow from the ones before, the gradients it left and the state before."""
    from idc_models_amd.engine import AdamW
    opt = AdamW(1e-3, weight_decay=0.05, global_clipnorm=clip, decay=decay, state_bits=bits)
    m = model(opt, arch)
    assert type(m.impl).__name__ == "FusedStep"
    x, y = batch()
    mask = mask_of(m, decay)
    for t in range(1, 5):
        w0, (m0, v0) = m.arena.data.double().cpu(), values(opt)
        loss, _ = m.impl.train_step(x, y)
        torch.cuda.synchronize()
        prog = next(iter(m.impl.progs.values()))
        assert not prog.host_optimizer and prog.opt_index is not None
        g = m.arena.grad.double().cpu()
        assert math.isfinite(loss.item()) and bool((opt.steps == t).all())
        w1, m1, v1, root, tw, tm, tv, tr = orc.step(w0, g, m0, v0, t, 1e-3, 0.9, 0.999, 1e-7, 0.05, mask, 1.0, clip or 0.0,
                                                    float(g.norm()))
        orc.within(m.arena.data, w1, tw)
        if bits == 32:
            orc.within(opt.m, m1, tm)
            orc.within(opt.v, v1, tv)
        else:
            _, high = orc.hash_bits(root.numel(), t)
            lo, hi, open_ = orc.code_bounds(root, 4, high, 16 * orc.U)
            have = values(opt)[1].sqrt()
            tiny = (root.view(-1, 64).amax(1) < 2.0 ** -62).repeat_interleave(64)
            assert bool(((have == lo) | (have == hi) | open_ | tiny).all())
    # set_lr reaches the replayed update
    prog.set_lr(0.0)
    w0 = m.arena.data.clone()
    m.impl.train_step(x, y)
    torch.cuda.synchronize()
    assert torch.equal(w0, m.arena.data) and int(opt.steps[0]) == 5


@pytest.mark.parametrize("bits", [32, 8])
def test_fused_skip_nonfinite(bits):
    from idc_models_amd.engine import AdamW
    opt = AdamW(1e-3, global_clipnorm=1.0, state_bits=bits)
    m = model(opt, skip_nonfinite=True)
    g = torch.Generator().manual_seed(1)
    x, y = torch.rand(8, 50, 50, 3, generator=g), torch.randint(0, 2, (8,), generator=g)
    m.impl.train_step(x, y)
    torch.cuda.synchronize()
    before = [m.arena.data.clone()] + [t.clone() for t in opt.state_tensors().values()]
    bad = x.clone()
    bad[0, 10, 10, 0] = float("inf")
    m.impl.train_step(bad, y)
    torch.cuda.synchronize()
    assert m.skipped_steps() == 1
    assert all(torch.equal(a, b) for a, b in zip(before, [m.arena.data] + list(opt.state_tensors().values())))
    m.impl.train_step(x, y)
    torch.cuda.synchronize()
    assert m.skipped_steps() == 1 and int(opt.steps[0]) == 2 and not torch.equal(before[0], m.arena.data)


def test_eager_backend_and_evaluation():
    """The eager backend calls the same kernels; evaluation leaves the state alone."""
    from idc_models_amd.engine import AdamW
    opt = AdamW(1e-3, weight_decay=0.0, state_bits=8, global_clipnorm=1.0)
    m = model(opt, arch="tinycnn", backend="eager")
    g = torch.Generator().manual_seed(2)
    x, y = torch.randint(0, 256, (16, 10, 10, 3), generator=g, dtype=torch.uint8), torch.randint(0, 2, (16,), generator=g)
    for t in (1, 2):
        w0, (m0, v0) = m.arena.data.double().cpu(), values(opt)
        m.impl.train_step(x, y)
        grad = m.arena.grad.double().cpu()
        w1, *_ , tw, _, _, _ = orc.step(w0, grad, m0, v0, t, 1e-3, 0.9, 0.999, 1e-7, 0.0, torch.zeros_like(w0), 1.0, 1.0, float(grad.norm()))
        orc.within(m.arena.data, w1, tw)
    state = [t.clone() for t in opt.state_tensors().values()]
    m.impl.eval_step(x, y)
    assert opt.iterations == 2 and all(torch.equal(a, b) for a, b in zip(state, opt.state_tensors().values()))


@pytest.mark.parametrize("bits", [32, 8])
def test_cpu_and_gpu_states_are_the_same_bits(bits):
    from idc_models_amd.engine import AdamW, ParamArena
    g = torch.Generator().manual_seed(4)
    shapes = [(3, 3, 16, 33), (33,), (500, 7), (1,)]
    init = [torch.randn(*s, generator=g) for s in shapes]
    arenas = [ParamArena([torch.nn.Parameter(t.clone().to(d)) for t in init]) for d in ("cpu", DEV)]
    opts = [AdamW(1e-2, state_bits=bits, decay="kernels") for _ in arenas]
    for o, a in zip(opts, arenas):
        o.bind(a)
    for t in range(1, 7):
        grad = torch.randn(arenas[0].numel, generator=g) * 10.0 ** (t % 4 - 3)
        for o, a in zip(opts, arenas):
            a.grad.copy_(grad)
            o.step(grad_scale=0.25)
    for k, v in opts[0].state_tensors().items():
        assert torch.equal(v, opts[1].state_tensors()[k].cpu()), k
    assert torch.allclose(arenas[0].data, arenas[1].data.cpu(), rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("width", [(32, 8), (8, 32), (8, 8)])
def test_checkpoint_resumes_on_the_gpu(tmp_path, width):
    """Resuming a run gives its next step's bits where the width is kept; of another width, the moments
    are the decoded (or rounded) ones."""
    from idc_models_amd.engine import AdamW
    x, y = batch()
    a = model(AdamW(1e-3, state_bits=width[0]), "vgg16")
    for _ in range(2):
        a.impl.train_step(x, y)
    path = str(tmp_path / "c.pt")
    a.save_checkpoint(path)
    b = model(AdamW(1e-3, state_bits=width[1]), "vgg16", seed=7)
    b.impl.train_step(x, y)
    b.load_checkpoint(path)
    torch.cuda.synchronize()
    assert torch.equal(a.arena.data, b.arena.data) and bool((b.optimizer.steps == 2).all())
    ma, va = values(a.optimizer)
    mb, vb = values(b.optimizer)
    for have, want in zip(b.optimizer.moments(), (mb, vb)):  # the kernel's decoding: r * r in fp32
        assert bool(((have.double().cpu() - want).abs() <= orc.U * want.abs() + 2.0 ** -149).all())
    if width[1] == 32 or width[0] == 8:
        assert torch.equal(ma, mb) and torch.equal(va, vb)
    else:
        top = ma.abs().view(-1, 64).amax(1).repeat_interleave(64)
        assert bool(((ma - mb).abs() <= ma.abs() / 16 * (1 + 1e-6) + top * 2.0 ** -17).all())
    if width[0] == 8 == width[1]:
        g = torch.randn_like(a.arena.grad)
        for m in (a, b):
            m.arena.grad.copy_(g)
            m.optimizer.step()
        assert torch.equal(a.arena.data, b.arena.data)
        assert all(torch.equal(p, q) for p, q in zip(a.optimizer.state_tensors().values(), b.optimizer.state_tensors().values()))


@pytest.mark.parametrize("bits", [32, 8])
def test_batched_clients_match_sequential(monkeypatch, bits):
    """Four federated clients with AdamW in one grouped program (each copy has its own moments, counter
    and norm) give bitwise the round of training them one after another."""
    from idc_models_amd.data import contiguous_clients, synthetic_dataset
    from idc_models_amd.engine import AdamW, Model
    from idc_models_amd.fed import build_federated_averaging_process
    from idc_models_amd.models import build_model
    from idc_models_amd.parallel import OneDeviceStrategy
    monkeypatch.setenv("IDC_DETERMINISTIC", "1")
    dev = torch.device("cuda", 0)
    base = build_model("densenet121", None, 1, seed=3)
    ds = synthetic_dataset(4 * 96, (50, 50, 3), 2, seed=7)

    def run(batching, rounds):
        clients = [c.batch(32, True, 1000, True, seed=k) for k, c in enumerate(contiguous_clients(ds, 4, 96))]
        proc = build_federated_averaging_process(
            lambda: Model(copy.deepcopy(base), OneDeviceStrategy(dev)),
            lambda: AdamW(1e-4, global_clipnorm=0.5, decay="kernels", state_bits=bits),
            lambda: AdamW(1e-3, weight_decay=0.0, state_bits=bits),
            average_bn_stats=True, backend="fused", client_batching=batching)
        state = proc.initialize()
        for _ in range(rounds):
            state, met = proc.next(state, clients)
        torch.cuda.synchronize()
        if batching:
            assert proc._grouped is not None and proc._grouped.k == 4
            steps = proc._grouped.region.view(proc._grouped.m.optimizer.steps)
            assert bool((steps == 3).all())  # every copy's every word: three batches of the last round
        return torch.cat([w.reshape(-1) for w in state.model.trainable]), state

    for rounds in (1, 2):
        a, sa = run(False, rounds)
        b, sb = run(True, rounds)
        assert torch.equal(a, b), float((a - b).abs().max())
        assert all(torch.equal(sa.optimizer_state[k], sb.optimizer_state[k]) for k in sa.optimizer_state)
        assert int(sa.optimizer_state["step"][0]) == rounds


@pytest.mark.parametrize("clip", [0.7, 0.013, 3.1])
@pytest.mark.parametrize("bits", [32, 8])
def test_cpu_and_gpu_states_are_the_same_bits_when_clipped(bits, clip):
    """Clip norms that are no powers of two, the gradients' norm above and below them; a table that its step sums
    by itself, and one with partial sums."""
    from idc_models_amd.engine import AdamW, ParamArena
    for shapes in ([(9, 11), (11,)], [(200, 300), (300,), (1,)]):
        g = torch.Generator().manual_seed(6)
        init = [torch.randn(*s, generator=g) for s in shapes]
        arenas = [ParamArena([torch.nn.Parameter(t.clone().to(d)) for t in init]) for d in ("cpu", DEV)]
        opts = [AdamW(1e-2, state_bits=bits, global_clipnorm=clip) for _ in arenas]
        for o, a in zip(opts, arenas):
            o.bind(a)
        for t in range(1, 13):
            grad = torch.randn(arenas[0].numel, generator=g) * 10.0 ** (t % 5 - 3)
            for o, a in zip(opts, arenas):
                a.grad.copy_(grad)
                o.step(grad_scale=0.3)
            for k, v in opts[0].state_tensors().items():
                assert torch.equal(v, opts[1].state_tensors()[k].cpu()), (k, t)


def test_cpu_and_gpu_codes_of_negative_zeros():
    """Gradients of -0.0 (as a masked backward leaves) that meet first moments which have rounded to -0: the CPU's
    codes, signs of zeros among them, are the GPU's."""
    from idc_models_amd.engine import AdamW, ParamArena
    arenas = [ParamArena([torch.nn.Parameter(torch.ones(64 * 6, device=d))]) for d in ("cpu", DEV)]
    opts = [AdamW(1e-2, state_bits=8) for _ in arenas]
    for o, a in zip(opts, arenas):
        o.bind(a)
    first = torch.full((384,), -1e-12)
    first[::64] = 1.0  # the others' values are far below a unit of their block
    first[320:] = -0.0
    zeros = torch.where(torch.arange(384) % 3 == 0, 0.0, -0.0)
    seen = 0
    for grad in (first, zeros, zeros, -zeros, zeros):
        for o, a in zip(opts, arenas):
            a.grad.copy_(grad)
            o.step()
        for k, v in opts[0].state_tensors().items():
            assert torch.equal(v, opts[1].state_tensors()[k].cpu()), k
        seen += int((opts[0].m == 0x80).sum())
    assert seen > 300
    # a checkpoint of the other width keeps them as well
    m, v = opts[1].moments()
    opts[0].load_slots({"m": m.cpu(), "v": v.cpu(), "step": opts[0].steps})
    assert torch.equal(opts[0].m, opts[1].m.cpu()) and torch.equal(opts[0].scales, opts[1].scales.cpu())


@pytest.mark.parametrize("bits,clip", [(32, None), (8, 0.1)])
def test_fused_update_is_adamw_(bits, clip):
    """The fused program's update gives the bits of adamw_ on the same gradients, also after set_lr; learning rates
    and decays whose product in fp32 is not the rounded product."""
    import numpy as np
    from idc_models_amd.engine import AdamW
    from idc_models_amd.ops import optim
    lr, wd = 1e-3, 0.004
    opt = AdamW(lr, weight_decay=wd, global_clipnorm=clip, state_bits=bits)
    m = model(opt, "mobilenetv2")
    x, y = batch()
    for t in range(4):
        assert np.float32(lr) * np.float32(wd) != np.float32(lr * wd)
        w = m.arena.data.clone()
        state = {k: v.clone() for k, v in opt.state_tensors().items()}
        m.impl.train_step(x, y)
        torch.cuda.synchronize()
        table = optim.TensorTable([m.arena.grad], [w])
        st = optim.AdamWState(table, bits=bits)
        for k, v in st.tensors().items():
            v.copy_(state[k])
        optim.adamw_(table, st, lr, weight_decay=wd, clip_norm=clip or 0.0)
        assert torch.equal(w, m.arena.data)
        assert all(torch.equal(v, opt.state_tensors()[k]) for k, v in st.tensors().items())
        if t == 1:
            lr = 3e-4
            next(iter(m.impl.progs.values())).set_lr(lr)


def test_clients_with_a_host_optimizer_train(monkeypatch):
    """SGD clients under client batching: the same round as one after another (they do not share a program, which
    would leave their weights as they were)."""
    from idc_models_amd.data import contiguous_clients, synthetic_dataset
    from idc_models_amd.engine import SGD, Model
    from idc_models_amd.fed import build_federated_averaging_process
    from idc_models_amd.models import build_model
    from idc_models_amd.parallel import OneDeviceStrategy
    monkeypatch.setenv("IDC_DETERMINISTIC", "1")
    base = build_model("vgg16", None, 1, seed=3)
    ds = synthetic_dataset(2 * 32, (50, 50, 3), 2, seed=7)

    def run(batching):
        clients = [c.batch(16, True, 1000, True, seed=k) for k, c in enumerate(contiguous_clients(ds, 2, 32))]
        proc = build_federated_averaging_process(lambda: Model(copy.deepcopy(base), OneDeviceStrategy(DEV)),
                                                 lambda: SGD(0.05), backend="fused", client_batching=batching)
        s0 = proc.initialize()
        s1, _ = proc.next(s0, clients)
        return [torch.cat([w.reshape(-1) for w in s.model.trainable]) for s in (s0, s1)]

    (a0, a1), (b0, b1) = run(False), run(True)
    assert torch.equal(a0, b0) and torch.equal(a1, b1) and not torch.equal(a0, a1)
