"""TensorTable's refusals and piece records, and the 8-bit moment codes, on the CPU."""
import math

import numpy as np
import pytest
import torch

from idc_models_amd.ops import moments8, optim

from . import adamw_oracle as orc


def t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def refused(match, grads, params=None, **kw):
    with pytest.raises(ValueError, match=match):
        optim.TensorTable(grads, params, **kw)


def test_refusals():
    refused("at least one", [])
    refused("dense tensors", [t(4).to_sparse()])
    refused("dense tensors", [None])
    refused("float32 or all bfloat16", [t(4, dtype=torch.float16)])
    refused("float32 or all bfloat16", [t(4), t(4, dtype=torch.bfloat16)])
    refused("one device", [t(4)], [t(4).to("meta")])
    refused("gaps", [t(4, 4)[:, :2]])
    refused("gaps", [t(4).expand(3, 4)])
    refused("gaps", [t(3, 4)], [t(4).expand(3, 4)])
    refused("needs params", [t(4)], decay=[True])
    refused("2 params for 1 grads", [t(4)], [t(4), t(4)])
    refused("params have to be float32", [t(4)], [t(4, dtype=torch.bfloat16)])
    refused("differ in shape", [t(4)], [t(5)])
    refused("differ in shape", [t(4, 3)], [t(3, 4).t()])
    refused("decay flags", [t(4)], [t(4)], decay=[True, False])
    p = t(100)
    refused("params overlap", [t(60), t(60)], [p[:60], p[40:]])
    refused("params overlap", [t(100), t(100)], [p, p])
    refused("params and grads overlap", [p[10:20]], [p[15:25]])
    refused("params and grads overlap", [t(100), p[3:5]], [p, t(2)])
    # fine but for the device: neighbours, a gradient that is used twice, empty tensors, permuted axes
    refused("on a GPU", [t(50), t(50)], [p[:50], p[50:]])
    g = t(50)
    refused("on a GPU", [g, g], [p[:50], p[50:]])
    refused("on a GPU", [t(0), t(5)], [t(0), t(5)])
    refused("on a GPU", [t(3, 4).t()], [t(3, 4).t()])
    refused("on a GPU", [t(4, dtype=torch.bfloat16)])


def test_refused_hyperparameters():
    ok = dict(lr=1e-3, beta_1=0.9, beta_2=0.999, epsilon=1e-7, weight_decay=0.0, clip_norm=0.0)
    optim.check_adamw(**ok)
    for k, v in (("beta_1", 1.0), ("beta_1", -0.1), ("beta_2", 1.0), ("beta_2", math.nan), ("lr", -1.0), ("lr", math.inf),
                 ("lr", math.nan), ("epsilon", -1e-9), ("epsilon", 0.0), ("epsilon", 1e-39), ("epsilon", math.nan), ("epsilon", 1e39), ("weight_decay", -1.0), ("clip_norm", -1.0), ("clip_norm", math.inf), ("clip_norm", 1e-40),
                 ("clip_norm", math.nan), ("lr", 1e39)):
        with pytest.raises(ValueError):
            optim.check_adamw(**dict(ok, **{k: v}))


def test_pieces_cover_every_element_once():
    sizes = [0, 1, 64, 65, 2047, 2048, 2049, 10 * 2048 + 1, 0]
    for grad_bytes, chunk in ((4, 2048), (2, 2048), (4, 4096)):
        w = np.cumsum([4096] + [4 * n + 4096 for n in sizes[:-1]]) // 16 * 16 + 4 * np.arange(len(sizes)) % 3
        g = np.cumsum([1 << 20] + [grad_bytes * n + 64 for n in sizes[:-1]]) // 16 * 16
        pieces, offsets, numel = optim.chunk_table(sizes, w, g, grad_bytes, [i % 2 == 0 for i in range(len(sizes))], chunk)
        assert offsets.tolist() == np.concatenate([[0], np.cumsum([orc.pad64(n) for n in sizes])[:-1]]).tolist()
        assert numel == sum(orc.pad64(n) for n in sizes)
        k = 0
        for i, n in enumerate(sizes):
            at = 0
            while at < n:
                c = pieces[k]
                assert c["w"] == w[i] + 4 * at and c["g"] == g[i] + grad_bytes * at and c["base"] == offsets[i] + at
                assert c["n"] == min(chunk, n - at) and c["base"] % 64 == 0
                assert bool(c["flags"] & 1) == (i % 2 == 0)
                assert bool(c["flags"] & 2) == (w[i] % 16 == 0 and g[i] % 16 == 0)
                assert c["base"] + orc.pad64(int(c["n"])) <= numel
                at += int(c["n"])
                k += 1
        assert k == len(pieces)


@pytest.mark.parametrize("mantissa", [moments8.M_BITS, moments8.ROOT_BITS])
def test_codes_are_decoded_exactly(mantissa):
    codes = torch.arange(256, dtype=torch.uint8)
    scales = torch.tensor([1, 100, 200, 254 - 30], dtype=torch.uint8)
    want = orc.code_values(codes, scales, mantissa)
    got = moments8.decode(codes, scales, mantissa)
    assert torch.equal(got.double(), want)
    assert torch.equal(got.bfloat16().double(), want)  # at most 5 significant bits
    again, s = moments8.encode(got, mantissa)
    assert torch.equal(orc.code_values(again, s, mantissa), want)
    assert bool(torch.isnan(moments8.decode(codes[:64], torch.tensor([255], dtype=torch.uint8), mantissa)).all())


@pytest.mark.parametrize("mantissa", [moments8.M_BITS, moments8.ROOT_BITS])
def test_dithered_codes_match_the_oracle(mantissa):
    g = torch.Generator().manual_seed(mantissa)
    x = torch.randn(64 * 500, generator=g) * 10.0 ** (torch.rand(64 * 500, generator=g) * 8 - 8)
    x[:64] = 0.0
    x[64] = 1e-30
    x[64:128] = torch.where(torch.arange(64) == 5, 3.0, 1e-30)
    if mantissa == moments8.ROOT_BITS:
        x = x.abs()
    low, high = moments8.dither(x.numel(), 17)
    a, b = orc.hash_bits(x.numel(), 17)
    assert torch.equal(low.long(), a) and torch.equal(high.long(), b)
    codes, scales = moments8.encode(x, mantissa, low)
    have = orc.code_values(codes, scales, mantissa)
    # y + one rounds y to 2^-24 of the binade: two roundings
    lo, hi, open_ = orc.code_bounds(x.double(), mantissa, a, 4 * orc.U)
    assert bool(((have == lo) | (have == hi) | open_).all())


def test_dither_is_even():
    """Over all 65536 values of the random bits a code's mean is the value, to 2^-16 of a step."""
    bits = torch.arange(65536, dtype=torch.int32)
    for mantissa in (moments8.M_BITS, moments8.ROOT_BITS):
        top = (2 ** (mantissa + 1) - 1) * 2.0 ** 14
        for value in (0.3, 5.75, 9.1, 100.3, 12345.678):
            blocks = torch.zeros(65536, 64)
            blocks[:, 0] = top  # sets the unit to 1
            blocks[:, 1] = value
            r = torch.zeros(65536, 64, dtype=torch.int32)
            r[:, 1] = bits
            codes, scales = moments8.encode(blocks.view(-1), mantissa, r.view(-1))
            assert bool((scales == 127).all())
            got = moments8.decode(codes, scales, mantissa).view(65536, 64)[:, 1].double()
            step = 2.0 ** max(math.floor(math.log2(value)) - mantissa, 0)
            if mantissa == moments8.ROOT_BITS and value < 1:
                assert bool((got == 1.0).all())  # a root keeps a code that is not zero
            else:
                assert abs(float(got.mean()) - value) <= step * 2.0 ** -15


def test_block_with_a_value_that_is_not_finite():
    for bad in (math.nan, math.inf, -math.inf):
        x = torch.ones(192)
        x[70] = bad
        codes, scales = moments8.encode(x, moments8.M_BITS)
        v = moments8.decode(codes, scales, moments8.M_BITS)
        assert bool(torch.isnan(v[64:128]).all()) and bool((v[:64] == 1).all()) and bool((v[128:] == 1).all())
        assert bool((codes[64:128] == 0).all())


def test_memory_at_held_addresses():
    """Replacing a tensor's storage leaves the memory of the first one alive, and is seen."""
    p, q = torch.nn.Parameter(torch.ones(1000)), torch.zeros(10)
    at = p.data_ptr()
    held = optim._Held([q, p])
    assert not held.moved() and not optim._Held([]).moved()
    with torch.no_grad():
        p.add_(1.0)
        p.grad = torch.zeros(1000)
    assert not held.moved()
    p.data = torch.full((1000,), 5.0)
    assert held.moved()
    others = [torch.full((1000,), 7.0) for _ in range(20)]  # none of them gets the first storage
    first = torch.empty(0).set_(held.memory[1])
    assert first.data_ptr() == at and bool((first == 2.0).all()) and first.numel() == 1000
    assert all(t.data_ptr() != at for t in others)
    p.data = first
    assert not held.moved()
    net = torch.nn.Linear(3, 4)
    held = optim._Held(list(net.parameters()))
    net.to(torch.float32)
    assert not held.moved()
    net.to(torch.float64)
    assert held.moved()


def test_zeros_keep_their_sign():
    """A first moment of -0.0 is code 0x80, as the kernel writes it, and stays so when it is decoded and encoded; a
    block that is not finite holds no signs."""
    x = torch.ones(128)
    x[1], x[2], x[3], x[4], x[70] = -0.0, 0.0, -1e-30, -1.0, -2.0
    codes, scales = moments8.encode(x, moments8.M_BITS)
    assert codes[:5].tolist() == [codes[0], 0x80, 0, 0x80, int(codes[0]) | 0x80]
    m = moments8.decode(codes, scales, moments8.M_BITS)
    assert torch.signbit(m).nonzero().flatten().tolist() == [1, 3, 4, 70]
    again, _ = moments8.encode(m, moments8.M_BITS)
    assert torch.equal(again, codes)
    x[100] = float("nan")
    codes, _ = moments8.encode(x, moments8.M_BITS)
    assert bool((codes[64:] == 0).all()) and codes[1] == 0x80


def test_state_of_other_tensors_is_refused():
    """Tables of [100, 30] and [30, 100] have states of one length, with other tensors' moments in it."""
    from types import SimpleNamespace
    dev = torch.device("cpu")
    table = lambda sizes: SimpleNamespace(params=[], sizes=list(sizes), numel=192, device=dev, _leaves=None)
    state = SimpleNamespace(sizes=[100, 30], numel=192, device=dev)
    for sizes in ([30, 100], [100, 31], [128, 64], [192], [100, 30, 0]):
        with pytest.raises(ValueError, match="another table"):
            optim.adamw_(table(sizes), state, 1e-3)
    with pytest.raises(ValueError, match="skip"):  # the same sizes: on to the next check
        optim.adamw_(table([100, 30]), state, 1e-3, skip=torch.zeros(1))


def test_autograd_is_told_of_changes():
    w, x = torch.nn.Parameter(torch.ones(5)), torch.ones(5, requires_grad=True)
    with torch.inference_mode():
        other = torch.zeros(3)  # has no version
    held = optim._Held([w, other])
    y = (w * x).sum()
    y.backward(retain_graph=True)
    held.changed()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    (w * x).sum().backward()
    optim._Held([]).changed()
