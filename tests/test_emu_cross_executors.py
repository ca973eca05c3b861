"""Encoder states of several tokens, as executors, their half clones and recordings share them, on the host emulator."""
import pytest
import torch

from test_emu_cross_states import BF16, engine  # noqa: F401  (the fixture)

LOC = "down_blocks.0.attentions.0"
ROWS = 6


def _half(eng, half):
    e = eng.clone_for_half(half)
    e.lib = e.run.lib = eng.lib  # the emulated library
    return e


def _attend(eng, h):
    """attn2 of one transformer: h [B, ROWS, 320] -> the same, as bits"""
    hid = h.clone().view(-1, 320)
    eng._cross_attention(LOC, hid, h.shape[0])
    return hid.view(h.shape)


@pytest.mark.parametrize("before,after", [("mask", None), (None, "mask"), ("mask", "mask"), ("mask", "other length"), (None, "other length")])
def test_half_executors_see_new_states_and_their_mask(engine, before, after):  # noqa: F811
    """states and mask set after the clones were made: each half computes what the whole batch's executor computes"""
    eng = engine[0]
    g = torch.Generator().manual_seed(11)
    h = torch.randn(2, ROWS, 320, generator=g).to(BF16)

    def states(kind):
        tokens = 7 if kind == "other length" else 5
        mask = None
        if kind is not None:
            mask = torch.rand(2, tokens, generator=g) < 0.5
            mask[:, 0], mask[:, 1] = True, False
        eng.set_encoder_hidden_states(torch.randn(2, tokens, 768, generator=g), mask)

    states(before)
    halves = [_half(eng, i) for i in (0, 1)]
    for i, e in enumerate(halves):
        assert torch.equal(_attend(e, h[i:i + 1]), _attend(eng, h)[i:i + 1])
    states(after)
    want = _attend(eng, h)
    for i, e in enumerate(halves):
        assert torch.equal(_attend(e, h[i:i + 1])[0], want[i]), i
    eng.set_encoder_hidden_states(torch.randn(2, 1, 768, generator=g))  # one token: no states, no mask, in any of them
    assert all(not e.cross_kv and e.cross_mask is None for e in (eng, *halves))
