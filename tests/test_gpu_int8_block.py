"""Whole encoder blocks with the products in 8-bit integers, against the float64 oracle.

Bar. Quantising a token row costs a noise of s / sqrt(12) per value, s = max / 127: for rows of 1024
or 4096 values of a bell-shaped distribution max is 3 to 5 deviations, so 0.7 to 1.1 % of the row's rms; requantising the
Q8_0 weights per channel costs as much again (their blocks' scales differ by up to four within a
channel, so up to 1.1 %). A linear is therefore off by up to 1.6 % rms, a branch of two linears by up to 2.3 % plus
what its non-linearities pass on (SiLU and GLU have slopes up to 1.1, the softmax and LayerNorm about
1), and a block adds four branches, with independent errors, to a stream that the branches make up: 2 x 2.3 % = 4.6 %
of the output's rms at most; two blocks sqrt(2) times that. The bars are 5 % and 7 %; a linear left out, doubled
or wired wrongly is off by tens of per cent.
"""
import numpy as np
import pytest
import torch

from oracle import block as ob
from oracle import int8 as oi
from parakeet_cuda_b200.block import EncoderBlocks
from parakeet_cuda_b200.layers import LAYER_PLAN
from parakeet_cuda_b200.pq8 import EPI_GLU, EPI_RESIDUAL, EPI_SILU
from parakeet_cuda_b200.runtime import Runtime
from parakeet_cuda_b200.synthetic import SyntheticParakeet

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def rt():
    return Runtime(0)


@pytest.fixture(scope='module')
def model():
    return SyntheticParakeet(seed=31, encoder_layers=2, decoder=False, block=True)


@pytest.mark.parametrize('windows,t,layers', [(1, 1, 1), (3, 33, 1), (2, 375, 1), (2, 60, 2)])
def test_int8_blocks_match_oracle(rt, model, windows, t, layers):
    x = np.random.default_rng(t).normal(size=(windows * t, 1024)).astype(np.float32)
    xd = torch.from_numpy(x).cuda()
    blocks = EncoderBlocks(model, rt, windows, t, layers=layers, products='int8')
    got = blocks.forward(xd).clone()
    gold = ob.blocks(x, model, list(range(layers)), windows=windows)
    err = np.sqrt(((got.double().cpu().numpy() - gold) ** 2).mean() / (gold ** 2).mean())
    print(f'{windows} x {t}, {layers} layer(s): rms error {err:.2e}')
    assert err <= (0.05 if layers == 1 else 0.07)
    # the same bits again, and from a captured graph
    assert torch.equal(blocks.forward(xd), got)
    blocks.buf['x'].copy_(xd)
    graph = blocks.capture()
    for _ in range(2):
        blocks.buf['x'].copy_(xd)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(blocks.buf['x'], got)
    assert rt.device_status() == 0


def test_int8_blocks_refuse(rt, model):
    with pytest.raises(ValueError):
        EncoderBlocks(model, rt, 1, 4, layers=1, products='int4')


def test_int8_block_linears(rt, model, monkeypatch):
    """Every linear of a block on what it really gets: the integers and the product of the oracle, with the
    oracle's requantised weights. (Its input's quotients are none within 1e-9 of a border where a norm comes
    first; plain rows have no such exception.) The bound is the product's: 4 U (|acc s t|) before the activation, U = 2^-24, a
    slope of at most 1.1, 8 U of the result for the activation, U for the residual's sum, half a step of the type."""
    u = 2.0 ** -24
    windows, t = 2, 33
    names = {}
    blocks = EncoderBlocks(model, rt, windows, t, layers=1, products='int8')
    for name, keys, *_ in LAYER_PLAN:
        w8 = blocks.linears[0][name]
        plain = np.concatenate([np.asarray(model.array(f'encoder.layers.0.{key}.weight'), np.float64).reshape(-1, w8.k) for key in keys])
        wq, ws, _ = oi.quantize(plain)
        assert np.array_equal(w8.q.cpu().numpy(), wq) and np.array_equal(w8.scale.cpu().numpy(), ws), name
        names[id(w8)] = name
    calls = []
    linear = Runtime.linear_i8

    def spy(self, x, w, out=None, bias=None, resid=None, epilogue=0, alpha=1.0, norm=None, out_dtype=None):
        kept = [x.clone(), None if resid is None else resid.clone()]
        y = linear(self, x, w, out=out, bias=bias, resid=resid, epilogue=epilogue, alpha=alpha, norm=norm, out_dtype=out_dtype)
        calls.append((names[id(w)], w, kept[0], kept[1], epilogue, alpha, norm, y.clone()))
        return y

    monkeypatch.setattr(Runtime, 'linear_i8', spy)
    blocks.forward(torch.from_numpy(np.random.default_rng(5).normal(size=(windows * t, 1024)).astype(np.float32)).cuda())
    assert [c[0] for c in calls] == [e[0] for e in LAYER_PLAN]
    f64 = lambda a: a.double().cpu().numpy()
    for name, w, x, resid, epilogue, alpha, norm, y in calls:
        h = f64(x) if norm is None else oi.layer_norm(f64(x), f64(norm[0]), f64(norm[1]))
        q, s, margin = oi.quantize(h)
        assert norm is None or margin.min() > 1e-9, name
        z, size = oi.product(q, s, w.q.cpu().numpy(), w.scale.cpu().numpy())
        err = 4 * u * size
        if epilogue == EPI_GLU:
            half = z.shape[1] // 2
            a, g, da, dg = z[:, :half], oi.sigmoid(z[:, half:]), err[:, :half], err[:, half:]
            want, err = a * g, da * g + np.abs(a) * 0.25 * dg + da * dg
        elif epilogue == EPI_RESIDUAL:
            want, err = f64(resid) + alpha * z, alpha * err
        else:
            want = oi.act(z, 'silu' if epilogue == EPI_SILU else 'none')
            err = 1.1 * err
        err = err + 8 * u * np.abs(want)
        err = err + torch.finfo(y.dtype).eps / 2 * (np.abs(want) + err) + 1e-37
        assert (np.abs(f64(y) - want) <= err).all(), (name, float((np.abs(f64(y) - want) / err).max()))


def test_int8_block_inputs_keep_their_bits(rt, model):
    """What the 8-bit products quantise has not been rounded to TF32 first: positions, attention and convolution outputs
    keep their low 13 bits (random ones are all 0 once in 8192)."""
    blocks = EncoderBlocks(model, rt, 2, 40, layers=1, products='int8')
    blocks.forward(torch.from_numpy(np.random.default_rng(6).normal(size=(80, 1024)).astype(np.float32)).cuda())
    for name, held in (('pos', blocks.pe), ('ctx', blocks.buf['ctx']), ('dw', blocks.buf['dw'])):
        low = held.contiguous().view(torch.int32) & 0x1FFF
        assert (low != 0).float().mean() > 0.5, name
    plain = np.asarray(model.array('encoder.pos_enc.pe'), np.float32)
    limit = int(model.metadata['asr.encoder.pos_emb_max_len'])
    assert np.array_equal(blocks.pe.cpu().numpy(), plain[limit - 40:limit + 39])
    tf32 = EncoderBlocks(model, rt, 2, 40, layers=1)
    assert not (tf32.pe.contiguous().view(torch.int32) & 0x1FFF).any()
