"""The language model without the feed-forward block is the one that it was
before there was a block, and with it differs by the block alone."""
import pytest
import torch
from torch import nn

from gtopkssgd_amd import models as zoo

KEYS = ["encoder.weight"] + [
    f"rnn.{kind}_l{layer}" for layer in (0, 1)
    for kind in ("weight_ih", "weight_hh", "bias_ih", "bias_hh")] + [
    "decoder.weight", "decoder.bias"]


def drawn(vocab, hidden):
    """The parameters, drawn layer by layer in the model's order."""
    enc = nn.Embedding(vocab, hidden)
    rnn = nn.LSTM(hidden, hidden, 2, dropout=0.65)
    nn.Linear(hidden, vocab)
    nn.init.uniform_(enc.weight, -0.1, 0.1)
    out = {"encoder.weight": enc.weight, "decoder.weight": enc.weight,
           "decoder.bias": torch.zeros(vocab)}
    out.update({f"rnn.{k}": v for k, v in rnn.state_dict().items()})
    return out


@pytest.mark.parametrize("ffn", [{}, {"ffn_mult": 0}, {"ffn_mult": 2},
                                 {"ffn_mult": 1, "act8": True}])
def test_parameters(ffn):
    torch.manual_seed(5)
    want = drawn(60, 16)
    torch.manual_seed(5)
    net = zoo.create_net("lstm", "ptb", vocab_size=60, hidden=16, **ffn)
    state = net.state_dict()
    own = [k for k in state if not k.startswith("ffn.")]
    assert own == KEYS
    assert bool(ffn.get("ffn_mult")) == (len(own) < len(state))
    assert all(torch.equal(state[k], want[k]) for k in KEYS)


def test_output():
    torch.manual_seed(5)
    net = zoo.lstm_ptb(60, 16).eval()
    toks = torch.randint(0, 60, (7, 3))
    got, hidden = net(toks, net.init_hidden(3))
    out, last = net.rnn(net.encoder(toks), net.init_hidden(3))
    want = nn.functional.linear(out, net.encoder.weight, net.decoder.bias)
    assert torch.equal(got, want)
    assert all(torch.equal(a, b) for a, b in zip(hidden, last))
