"""The label decoder's sampled answers (lib/lstm/decoder_rnn.py, DecoderRNN.sampling) where nothing can be drawn."""
import math

import pytest
import torch
from torch.nn.utils.rnn import PackedSequence

pytestmark = pytest.mark.gpu

N, H = 6, 64


@pytest.fixture()
def decoder():
    from lib.lstm.decoder_rnn import DecoderRNN
    torch.manual_seed(3)
    classes = ['__background__'] + ['person', 'dog', 'cat', 'tree', 'car', 'hat', 'shoe', 'window', 'table', 'plate']
    return DecoderRNN(classes, embed_dim=100, inputs_dim=H, hidden_dim=H, recurrent_dropout_probability=0.0).cuda().eval()


def answers(decoder, x, **sampling):
    g = torch.Generator(device='cuda')
    g.manual_seed(5)
    decoder.sampling = dict(sampling, generator=g)
    with torch.no_grad():
        dists, labels = decoder(PackedSequence(x, torch.ones(x.shape[0], dtype=torch.long)))
    return dists, labels


@pytest.mark.parametrize('bias', ['nan', 'minus infinity'])
def test_a_row_that_cannot_be_drawn_from_gives_its_arg_max(decoder, bias):
    """never the background, which no step answers with"""
    with torch.no_grad():
        if bias == 'nan':
            decoder.out.bias[7] = math.nan
        else:
            decoder.out.bias[1:] = -math.inf
    x = torch.randn(N, H, generator=torch.Generator().manual_seed(1)).cuda()
    for sampling in (dict(), dict(temperature=0.0), dict(temperature=2.0, top_k=4, top_p=0.9)):
        dists, labels = answers(decoder, x, **sampling)
        assert torch.equal(labels, dists[:, 1:].max(1)[1] + 1)
        assert int(labels.min()) >= 1


def test_the_rows_before_one_that_cannot_be_drawn_from(decoder):
    x = torch.randn(N, H, generator=torch.Generator().manual_seed(2)).cuda()
    _, want = answers(decoder, x, temperature=3.0)
    assert int(want.min()) >= 1
    x[3] = math.nan              # its state, and so every later one, is a NaN
    dists, labels = answers(decoder, x, temperature=3.0)
    assert bool(torch.isnan(dists[3:]).any(1).all()) and not bool(torch.isnan(dists[:3]).any())
    assert torch.equal(labels[:3], want[:3])
    assert torch.equal(labels[3:], dists[3:, 1:].max(1)[1] + 1)
