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


def test_a_recorded_step_keeps_its_scratch(engine, monkeypatch):  # noqa: F811
    """recorded without an eager pass before it: the scratch that one level's launches were recorded with is still there when another
    level has asked for more, and the replay computes what an eager pass does"""
    import ctypes

    from humanvid_amd import engine as E

    eng, sd, cfg = engine
    g = torch.Generator().manual_seed(13)
    tokens = 1100  # few queries, many states: ranges, joined through scratch
    shared = eng
    eng = _half(eng, 0)
    eng.cfg_half = None  # the whole batch, with a workspace that nothing has used
    levels = [("down_blocks.0.attentions.0", 320), ("mid_block.attentions.0", cfg["block_out_channels"][-1])]
    assert levels[1][1] > 320
    eng.locations = [loc for loc, _ in levels]
    shared.set_encoder_hidden_states(torch.randn(2, 2, 768, generator=g))  # (their weights)
    for loc, C in levels:  # what the projection of many tokens would leave here, without its time on the emulator
        eng.cross_kv[loc] = torch.randn(2, tokens, 2 * C, generator=g).to(BF16)
    hid = {loc: torch.randn(2 * ROWS, C, generator=g).to(BF16) for loc, C in levels}
    used, call = [], E.ops.cross_attention

    def logged(*a, workspace=None, **kw):
        if workspace is not None:
            used.append((workspace.data_ptr(), workspace.numel()))
        return call(*a, workspace=workspace, **kw)

    monkeypatch.setattr(E.ops, "cross_attention", logged)
    h = ctypes.c_void_p()
    eng.lib.call("hv_cmdlist_begin")
    try:
        for loc, _ in levels:
            eng._cross_attention(loc, hid[loc], 2)
    finally:
        eng.lib.call("hv_cmdlist_end", ctypes.byref(h))
    try:
        assert len(used) == 2 and used[0][1] < used[1][1]
        held = [(t.data_ptr(), t.numel()) for t in eng.ws.bufs.values()]
        for at, n in used:
            assert any(p <= at and at + 4 * n <= p + 4 * m for p, m in held), "scratch of the recording was let go"
        for kv in eng.cross_kv.values():  # new states in the same buffers
            kv.copy_(torch.randn(kv.shape, generator=g))
        want = {loc: torch.randn(t.shape, generator=g).to(BF16) for loc, t in hid.items()}
        for loc, t in hid.items():
            t.copy_(want[loc])
        eng.lib.call("hv_cmdlist_run", h, None)
        for loc, t in hid.items():
            eng._cross_attention(loc, want[loc], 2)
            assert torch.equal(t, want[loc]), loc
    finally:
        eng.lib.call("hv_cmdlist_destroy", h)
        shared.cross_kv.clear()


def test_states_narrower_than_the_packed_weights():
    """a model whose encoder states have 96 channels (its packed weights are padded to 128): one token and several"""
    from test_emu_engine import O, _engine_on_emulator
    from humanvid_amd.unet3d import UNet3DConditionModel

    cfg = O.tiny_unet3d_cfg(cross_attention_dim=96)
    sd = O.make_unet3d_weights(cfg, seed=2)
    net = UNet3DConditionModel(**dict(cfg, use_inflated_groupnorm=True, unet_use_cross_frame_attention=False,
                                      unet_use_temporal_attention=False, motion_module_type="Vanilla"))
    net.load_state_dict(sd, strict=True)
    eng, (hvlib, restore) = _engine_on_emulator(net)
    try:
        eng.locations = [LOC]
        t = LOC + ".transformer_blocks.0"
        heads = cfg["attention_head_dim"]
        g = torch.Generator().manual_seed(17)
        e = torch.randn(2, 3, 96, generator=g)
        eng.set_encoder_hidden_states(e[:, :1])
        want = torch.nn.functional.linear(torch.nn.functional.linear(e[:, 0], sd[t + ".attn2.to_v.weight"]),
                                          sd[t + ".attn2.to_out.0.weight"], sd[t + ".attn2.to_out.0.bias"])
        assert float((eng.cross_const[LOC].float() - want).norm() / want.norm()) < 1e-2  # bf16 weights and states
        eng.set_encoder_hidden_states(e)
        h = torch.randn(2, ROWS, 320, generator=g).to(BF16)
        got = _attend(eng, h)
        for b in range(2):
            want = h[b:b + 1].float() + O.attention(sd, t + ".attn2", O.layer_norm(sd, t + ".norm2", h[b:b + 1].float()), e[b:b + 1], heads)
            assert float((got[b].float() - want[0]).norm() / want.norm()) < 1e-2
        for width in (64, 128):
            for tokens in (1, 3):
                with pytest.raises(ValueError, match="96 channels"):
                    eng.set_encoder_hidden_states(torch.randn(2, tokens, width, generator=g))
    finally:
        hvlib.current_stream = restore


def test_frames_of_a_shard(engine):  # noqa: F811
    """an executor that holds some of the frames computes the rows that one with all of them does"""
    eng = engine[0]
    g = torch.Generator().manual_seed(19)
    mask = torch.rand(2, 9, generator=g) < 0.6
    mask[:, 0] = True
    eng.set_encoder_hidden_states(torch.randn(2, 9, 768, generator=g), mask)
    h = torch.randn(2, 3 * ROWS, 320, generator=g).to(BF16)  # three frames
    want = _attend(eng, h)
    for f0, f1 in ((0, 2), (2, 3)):
        assert torch.equal(_attend(eng, h[:, f0 * ROWS:f1 * ROWS]), want[:, f0 * ROWS:f1 * ROWS])


@pytest.mark.parametrize("tokens", [1, 4])
def test_states_of_too_few_entries_are_refused_before_anything_runs(engine, tokens, monkeypatch):  # noqa: F811
    """a forward of two batch entries with the states of one: the second entry's row lies behind the table"""
    from humanvid_amd import engine as E

    eng = engine[0]

    def launched(*a, **kw):
        raise AssertionError("a kernel was launched")

    def forward(e, B):
        return e.forward_nhwc(torch.zeros(2 * B, 8, 4, 32, dtype=BF16), torch.zeros(B), None, B=B, F=2)

    halves = [_half(eng, i) for i in (0, 1)]
    eng.cross_const.clear()  # (a table of this test's own: one row)
    eng.set_encoder_hidden_states(torch.randn(1, tokens, 768))
    monkeypatch.setattr(E.ops, "timestep_embedding", launched)  # the first kernel of a forward
    for e, B in ((eng, 2), (halves[1], 1)):
        with pytest.raises(ValueError, match="batch entries"):
            forward(e, B)
    for e in (eng, halves[0]):  # one entry: as far as the first kernel
        with pytest.raises(AssertionError, match="launched"):
            forward(e, 1)
