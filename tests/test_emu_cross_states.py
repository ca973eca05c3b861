"""Encoder states of several tokens in the native executor, on the host emulator: the cross attention of one transformer."""
import pytest
import torch

from test_emu_engine import O, _engine_on_emulator

BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def engine():
    from humanvid_amd.unet3d import UNet3DConditionModel

    cfg = O.tiny_unet3d_cfg()
    sd = O.make_unet3d_weights(cfg, seed=0)
    net = UNet3DConditionModel(**dict(cfg, use_inflated_groupnorm=True, unet_use_cross_frame_attention=False,
                                      unet_use_temporal_attention=False, motion_module_type="Vanilla"))
    net.load_state_dict(sd, strict=True)
    eng, (hvlib, restore) = _engine_on_emulator(net)
    try:
        yield eng, sd, cfg
    finally:
        hvlib.current_stream = restore


def _want(sd, t, h, ehs, heads):
    return h + O.attention(sd, t + ".attn2", O.layer_norm(sd, t + ".norm2", h), ehs, heads)


@pytest.mark.parametrize("tokens,masked", [(5, False), (33, True), (1, True)])
def test_transformer_attends_to_the_states(engine, tokens, masked):
    eng, sd, cfg = engine
    g = torch.Generator().manual_seed(tokens)
    B, rows = 2, 6
    ehs = torch.randn(B, tokens, 768, generator=g)
    mask = torch.rand(B, tokens, generator=g) < 0.6 if masked else None
    if masked:
        mask[0, 0], mask[1] = True, False  # the second entry attends to nothing
    eng.set_encoder_hidden_states(ehs, mask)
    loc = "down_blocks.0.attentions.0"
    t = loc + ".transformer_blocks.0"
    h = torch.randn(B, rows, 320, generator=g).to(BF16)
    hid = h.clone().view(B * rows, 320)
    eng._cross_attention(loc, hid, B)
    heads = cfg["attention_head_dim"]
    for b in range(B):
        if masked and not bool(mask[b].any()):
            want = h[b:b + 1].float() + sd[t + ".attn2.to_out.0.bias"]
        else:
            want = _want(sd, t, h[b:b + 1].float(), ehs[b:b + 1] if mask is None else ehs[b:b + 1, mask[b]], heads)
        err = float((hid.view(B, rows, 320)[b].float() - want[0]).norm() / want.norm())
        assert err < 1e-2, err  # bf16 weights, states, queries and output
    # an executor of the second half alone
    half = eng.clone_for_half(1)
    half.lib = half.run.lib = eng.lib
    hid1 = h[1:].clone().view(rows, 320)
    half._cross_attention(loc, hid1, 1)
    assert torch.equal(hid1, hid.view(B, rows, 320)[1])


def test_states_refusals_and_the_way_back(engine):
    eng, sd, cfg = engine
    e = torch.randn(2, 4, 768)
    with pytest.raises(ValueError):
        eng.set_encoder_hidden_states(e[0])
    with pytest.raises(ValueError):
        eng.set_encoder_hidden_states(e[:, :0])
    for tokens in (1, 4):
        with pytest.raises(ValueError, match="768 channels"):
            eng.set_encoder_hidden_states(e[:, :tokens, :512])
    with pytest.raises(ValueError):
        eng.set_encoder_hidden_states(e, torch.ones(2, 5))
    eng.set_encoder_hidden_states(e)
    with pytest.raises(ValueError):
        eng._cross_attention("down_blocks.0.attentions.0", torch.zeros(18, 320, dtype=BF16), 3)
    buffers = {k: v.data_ptr() for k, v in eng.cross_kv.items()}
    eng.set_encoder_hidden_states(torch.randn(2, 4, 768))  # another clip: the same buffers
    assert buffers == {k: v.data_ptr() for k, v in eng.cross_kv.items()}
    eng.set_encoder_hidden_states(e[:, :1])  # one token: the folded constant again
    assert not eng.cross_kv and eng.cross_mask is None and len(eng.cross_const) == len(eng.locations)
