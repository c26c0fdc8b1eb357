"""AdamW as the framework uses it, on the CPU: the optimizer, checkpoints, the FedAvg server, recipes."""
import copy

import pytest
import torch

from idc_models_amd.engine import AdamW, Model, ParamArena, optimizers
from idc_models_amd.models import build_model
from idc_models_amd.parallel import OneDeviceStrategy

from . import adamw_oracle as orc

CPU = OneDeviceStrategy("cpu")


def small_arena(seed=0):
    g = torch.Generator().manual_seed(seed)
    shapes = [(3, 3, 5, 7), (7,), (7,), (70, 3), (3,), (1,)]
    arena = ParamArena([torch.nn.Parameter(torch.randn(*s, generator=g)) for s in shapes])
    return arena, g


def fill(arena, g, scale):
    for p in arena.params:
        p.grad.copy_(torch.randn(p.shape, generator=g) * scale)


@pytest.mark.parametrize("decay", ["all", "kernels"])
@pytest.mark.parametrize("clip", [None, 0.5])
@pytest.mark.parametrize("bits", [32, 8])
def test_cpu_steps_match_the_formula(bits, clip, decay):
    arena, g = small_arena()
    opt = AdamW(1e-2, weight_decay=0.1, global_clipnorm=clip, decay=decay, state_bits=bits)
    opt.bind(arena)
    mask = torch.zeros(arena.numel, dtype=torch.float64)
    for p, s in zip(arena.params, arena.slots):
        mask[s.offset:s.offset + s.numel] = float(decay == "all" or p.dim() > 1)
    for t in range(1, 5):
        fill(arena, g, 10.0 ** (t - 3))
        w0, grad = arena.data.double(), arena.grad.double()
        if bits == 32:
            m0, v0 = opt.m.double(), opt.v.double()
        else:
            m0 = orc.code_values(opt.m, opt.scales[:, 0], 3)
            v0 = orc.code_values(opt.v, opt.scales[:, 1], 4) ** 2
        opt.step(grad_scale=0.5)
        w1, m1, v1, root, tw, tm, tv, _ = orc.step(w0, grad, m0, v0, t, 1e-2, 0.9, 0.999, 1e-7, 0.1, mask, 0.5, clip or 0.0,
                                                   orc.norm([arena.grad]))
        orc.within(arena.data, w1, tw)
        assert opt.iterations == t and bool((opt.steps == t).all())
        if bits == 32:
            orc.within(opt.m, m1, tm)
            orc.within(opt.v, v1, tv)
        else:
            low, high = orc.hash_bits(arena.numel, t)
            have = orc.code_values(opt.v, opt.scales[:, 1], 4)
            lo, hi, open_ = orc.code_bounds(root, 4, high, 16 * orc.U)
            assert bool(((have == lo) | (have == hi) | open_).all())
            # one step of the codes of m: 1/8 of the value, or a unit (2^-17 of the block's largest)
            top = m1.abs().view(-1, 64).amax(1).repeat_interleave(64)
            have = orc.code_values(opt.m, opt.scales[:, 0], 3)
            assert bool(((have - m1).abs() <= m1.abs() / 8 + top * 2.0 ** -16 + tm).all())


def test_refusals_and_names():
    for kw in (dict(state_bits=16), dict(decay="none"), dict(beta_1=1.0), dict(weight_decay=-1.0),
               dict(global_clipnorm=-1.0), dict(epsilon=float("nan"))):
        with pytest.raises(ValueError):
            AdamW(**kw)
    opt = optimizers.get("adamw")
    assert isinstance(opt, AdamW) and opt.native_step and opt.get_config()["state_bits"] == 32
    assert AdamW(lr=0.5).learning_rate == 0.5 and opt.state_tensors() == {}
    assert not optimizers.get("sgd").native_step and optimizers.get("rmsprop").native_step


def test_skip_nonfinite_and_reset():
    arena, g = small_arena()
    opt = AdamW(state_bits=8)
    opt.bind(arena)
    opt.skip_nonfinite = True
    fill(arena, g, 1.0)
    opt.step()
    before = [arena.data.clone()] + [t.clone() for t in opt.state_tensors().values()]
    arena.grad[3] = float("inf")
    opt.step()
    assert opt.skipped == 1 and all(torch.equal(a, b) for a, b in zip(before, [arena.data] + list(opt.state_tensors().values())))
    with pytest.raises(ValueError, match="bound to"):
        opt.step(small_arena()[0])
    opt.reset_state()
    assert all(int(t.abs().max() if t.dtype != torch.uint8 else t.max()) == 0 for t in opt.state_tensors().values())


def tiny(opt, seed=0):
    m = Model(build_model("tinycnn", seed=seed), CPU)
    m.compile(opt, "binary_crossentropy", ["accuracy"])
    return m


@pytest.mark.parametrize("width", [(32, 32), (8, 8), (32, 8), (8, 32)])
def test_checkpoints_of_either_width(tmp_path, width):
    from idc_models_amd.data import prepare_for_training, synthetic_dataset
    ds = synthetic_dataset(64, (10, 10, 3), seed=0)
    a = tiny(AdamW(1e-3, state_bits=width[0]))
    a.fit(prepare_for_training(ds, 16), epochs=1, verbose=0)
    path = str(tmp_path / "state.pt")
    a.save_checkpoint(path)
    b = tiny(AdamW(1e-3, state_bits=width[1]), seed=3)
    b.load_checkpoint(path)
    assert b.optimizer.iterations == 4 and bool((b.optimizer.steps == 4).all())
    (ma, va), (mb, vb) = a.optimizer.moments(), b.optimizer.moments()
    if width in ((32, 32), (8, 8), (8, 32)):  # codes are fp32 values
        assert torch.equal(ma, mb) and torch.equal(va, vb)
        return
    for x, y, step in ((ma, mb, 1 / 16), (va.sqrt(), vb.sqrt(), 1 / 32)):  # to the nearest: half a code's step
        top = x.abs().view(-1, 64).amax(1).repeat_interleave(64)
        unit = top * 2.0 ** (-17 if step == 1 / 16 else -18)
        # (a root keeps a code that is not zero: up to a unit off)
        assert bool(((x - y).abs() <= x.abs() * step * (1 + 1e-6) + unit).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_fedavg_server_adamw(bits, tmp_path):
    """The server's weights take AdamW steps along minus the mean delta; its moments travel in the
    server state, also through a file."""
    from idc_models_amd.data import contiguous_clients, synthetic_dataset
    from idc_models_amd.engine import RMSprop
    from idc_models_amd.fed import build_federated_averaging_process, load_server_state, save_server_state
    base = build_model("tinycnn", seed=1)
    clients = lambda: [c.batch(16, False) for c in contiguous_clients(synthetic_dataset(48, (10, 10, 3), seed=2), 3, 16)]

    def make(server):
        return build_federated_averaging_process(lambda: Model(copy.deepcopy(base), CPU), lambda: RMSprop(1e-2), server)

    def round_(proc, state):
        torch.manual_seed(5)  # the clients' dropout
        return proc.next(state, clients())[0]

    plain, adaptive = make(None), make(lambda: AdamW(1e-2, weight_decay=0.0, state_bits=bits))
    s0 = plain.initialize()
    mean = [(a - b).double() for a, b in zip(round_(plain, s0).model.trainable, s0.model.trainable)]
    s1 = round_(adaptive, s0)
    g, offs = orc.place([-d for d in mean])
    w0, _ = orc.place(s0.model.trainable)
    z = torch.zeros_like(g)
    w1, *_ = orc.step(w0, g, z, z, 1, 1e-2, 0.9, 0.999, 1e-7, 0.0, z)
    for w, o in zip(s1.model.trainable, offs):
        # the delta that SGD's result gives back carries the rounding of two weights, which the first step's
        # quotient g / |g| sees where the delta is as small as that
        want = w1[o:o + w.numel()].view(w.shape)
        big = (g[o:o + w.numel()].abs() > 1e-4).view(w.shape)
        assert float(((w.double() - want).abs() * big).max()) <= 1e-5
    assert int(s1.optimizer_state["step"][0]) == 1 and s0.optimizer_state == {}
    s2 = round_(adaptive, s1)
    path = str(tmp_path / "s.pt")
    save_server_state(s1, path)
    other = make(lambda: AdamW(1e-2, weight_decay=0.0, state_bits=bits))
    s2b = round_(other, load_server_state(path))
    assert int(s2.optimizer_state["step"][0]) == 2
    assert all(torch.equal(a, b) for a, b in zip(s2.model.trainable, s2b.model.trainable))
    assert all(torch.equal(s2.optimizer_state[k], s2b.optimizer_state[k]) for k in s2.optimizer_state)


def test_recipe_optimizers():
    from idc_models_amd.recipes.transfer import TransferConfig, make_optimizer
    cfg = TransferConfig(optimizer="adamw", optimizer_args={"weight_decay": 0.02, "state_bits": 8})
    opt = make_optimizer(cfg.optimizer, 1e-3, cfg.optimizer_args)
    assert isinstance(opt, AdamW) and opt.weight_decay == 0.02 and opt.state_bits == 8 and opt.learning_rate == 1e-3
    assert make_optimizer(TransferConfig().optimizer, 1e-3).name == "RMSprop"
    with pytest.raises(ValueError, match="adamw, rmsprop"):
        make_optimizer("adam", 1e-3)


def test_cli_trains_with_adamw(tmp_path, capsys):
    from idc_models_amd.cli import main
    cfg = tmp_path / "c.yaml"
    cfg.write_text("synthetic_size: 160\nbatch_size: 8\ninitial_epochs: 1\nfine_tune_epochs: 1\nvalidation_steps: 1\n"
                   "steps_per_epoch: 1\nplot: false\noptimizer_args: {state_bits: 8, global_clipnorm: 1.0, decay: kernels}\n")
    main(["dist", "mobile", str(tmp_path), "--synthetic", "--strategy", "one", "--config", str(cfg), "--optimizer", "adamw"])
    assert "Number of layers" in capsys.readouterr().out


def _replica(rank, world, kind, bits):
    from idc_models_amd.data import synthetic_dataset
    from idc_models_amd.parallel import CentralStorageStrategy, MirroredStrategy
    st = (MirroredStrategy if kind == "mirrored" else CentralStorageStrategy)(backend="gloo")
    torch.manual_seed(rank)  # dropout differs, what is reduced is one gradient
    m = Model(build_model("tinycnn", seed=3), st)
    m.compile(AdamW(1e-2, global_clipnorm=0.1, state_bits=bits), "binary_crossentropy", ["accuracy"], backend="eager")
    m.fit(synthetic_dataset(64, (10, 10, 3), seed=11).batch(16, drop_remainder=True), epochs=2, verbose=0)
    return m.arena.data.numpy().copy(), {k: t.numpy().copy() for k, t in m.optimizer.state_tensors().items()}


@pytest.mark.parametrize("kind,bits", [("mirrored", 8), ("mirrored", 32), ("central", 8)])
def test_replicas_stay_the_same(kind, bits):
    from idc_models_amd.parallel.launch import spawn
    (w0, s0), (w1, s1) = spawn(_replica, 2, (kind, bits))
    assert (w0 == w1).all() and (s0["step"] == 8).all()
    if kind == "mirrored":
        assert all((s0[k] == s1[k]).all() for k in s0)
    else:  # rank 0 owns the state
        assert (s1["step"] == 0).all() and (s1["m"] == 0).all() and (s0["m"] != 0).any()


def test_clipped_gradients_take_one_quotient():
    """The factor of clipped gradients is clip / norm rounded once, as the GPU's: the first step's moments are
    bits of (1 - beta_1) * (g * factor)."""
    import numpy as np
    f = np.float32
    for seed in range(40):
        g = torch.Generator().manual_seed(seed)
        arena = ParamArena([torch.nn.Parameter(torch.randn(50, 7, generator=g))])
        arena.grad.copy_(torch.randn(arena.numel, generator=g) * 3)
        opt = AdamW(1e-2, global_clipnorm=0.7)
        opt.bind(arena)
        opt.step(grad_scale=0.3)
        grad = arena.grad.numpy()
        norm = f(np.sqrt(np.square(grad.astype(np.float64)).sum())) * f(0.3)
        want = f(0.1) * ((grad * f(0.3)) * (f(0.7) / norm))
        assert want.dtype == f and (opt.m.numpy() == want).all(), seed


def test_client_batching_needs_an_optimizer_that_the_program_carries():
    """A grouped program updates its weights by itself: clients whose optimizer steps on the host train one after
    another."""
    from types import SimpleNamespace
    from idc_models_amd.data import contiguous_clients, synthetic_dataset
    from idc_models_amd.engine import SGD, RMSprop
    from idc_models_amd.fed.grouped import eligible
    sets = [c.batch(8, drop_remainder=True) for c in contiguous_clients(synthetic_dataset(32, (10, 10, 3), seed=2), 2, 16)]
    model = lambda opt: SimpleNamespace(device=torch.device("cuda"), impl=SimpleNamespace(name="fused"),
                                        net=SimpleNamespace(num_outputs=1), optimizer=opt)
    for opt in (RMSprop(), AdamW(), AdamW(state_bits=8)):
        assert eligible(sets, model(opt))
    for opt in (SGD(0.1), SGD(0.1, momentum=0.9), RMSprop(momentum=0.9), RMSprop(centered=True)):
        assert not eligible(sets, model(opt))


@pytest.mark.parametrize("bits", [32, 8])
def test_secure_clients_keep_their_adamw_state(bits):
    """Clients of a secure federated process share one model and optimizer, whose slots (moments, scales, step
    counter) are swapped: after two rounds each has the bits of a client with an optimizer of its own."""
    from idc_models_amd.data import shard_clients, synthetic_dataset
    from idc_models_amd.fed import SecureFederatedProcess
    ds = synthetic_dataset(48, (10, 10, 3), seed=3)
    sets = lambda: [(s.take(18).batch(6, False), s.skip(18).batch(6, False)) for s in shard_clients(ds, 2)]

    def make():
        return tiny(AdamW(1e-2, global_clipnorm=0.5, state_bits=bits))

    proc = SecureFederatedProcess(make, sets(), percent=1.0, mode="mask", epochs=2)
    own = [make() for _ in range(2)]
    for k, m in enumerate(own):
        with torch.no_grad():
            for t, w in zip(m.net.weights, proc.states[k].weights):
                t.copy_(w)
    data = sets()
    for r in range(2):
        for k, m in enumerate(own):
            torch.manual_seed(10 * r + k)  # dropout
            proc.client_fit(k)
            torch.manual_seed(10 * r + k)
            m.fit(data[k][0], epochs=2, validation_data=data[k][1], verbose=0)
            assert all(torch.equal(a, b) for a, b in zip(proc.states[k].weights, m.net.weights))
            slots = m.optimizer.state_tensors()
            assert set(slots) == set(proc.states[k].opt_slots) and int(slots["step"][0]) == 6 * (r + 1)
            assert all(torch.equal(v, proc.states[k].opt_slots[n]) for n, v in slots.items())
        avg = proc.aggregate()  # both take the mean, with their own moments
        for k, m in enumerate(own):
            proc.states[k].weights = [a.detach().clone() for a in avg]
            with torch.no_grad():
                for t, a in zip(m.net.weights, avg):
                    t.copy_(a)
