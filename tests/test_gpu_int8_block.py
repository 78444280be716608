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
from parakeet_cuda_b200.block import EncoderBlocks
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
