"""Encoder states of several tokens on a real MI355X: with reference banks and guidance, in the executors of the halves, in a recorded
step; the 8-bit product in ranges under graph replays and on two streams.

Tolerance against the oracle: that of the one-token forwards (tests/test_gpu_unet.py)."""
import pytest
import torch

import operator_edge_cases as ec
import test_gpu_unet as T
from humanvid_amd import ops
from test_gpu_operators import cx  # noqa: F401  (the fixture)

O = T.O
pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _problem(tokens, seed, f=4, hh=8, ww=8):
    cfg = O.tiny_unet3d_cfg()
    sd = O.make_unet3d_weights(cfg, seed=0)
    g = torch.Generator().manual_seed(seed)
    sample = torch.randn(1, 4, f, hh, ww, generator=g).repeat(2, 1, 1, 1, 1)
    ehs = torch.randn(2, tokens, 768, generator=g)
    pose = (torch.randn(1, 320, f, hh, ww, generator=g) * 0.5).repeat(2, 1, 1, 1, 1)
    banks = {p: torch.randn(2, hh * ww if sd[p + ".norm.weight"].numel() == 320 else hh * ww // 4, sd[p + ".norm.weight"].numel(),
                            generator=g).half().float() for p in O.transformer_locations(cfg)}
    return cfg, sd, g, sample, ehs, pose, banks


def test_a_prompt_with_banks_and_guidance():
    cfg, sd, g, sample, ehs, pose, banks = _problem(77, 31)
    net = T.build_native(cfg, sd)
    ref = O.unet3d_forward(sd, cfg, sample, 601, ehs, pose, banks, do_cfg=True)
    out = T.run_native(net, sample, 601, ehs, pose, banks)
    assert T.nrmse(out, ref) < T.TOL
    assert T.nrmse(T.run_native(net, sample, 601, ehs, pose, {k: -v for k, v in banks.items()}), ref) > 1e-2  # the banks matter
    # a mask of its own for each half
    mask = torch.zeros(2, 77, dtype=torch.bool)
    mask[0, :5], mask[1, 40:] = True, True
    net.engine().set_reference_banks({k: v.cuda() for k, v in banks.items()}, do_cfg=True)
    got = net(sample.cuda(), 601, ehs.cuda(), pose_cond_fea=pose.cuda(), return_dict=False, encoder_attention_mask=mask.cuda())[0]
    short = torch.cat([ehs[:1, :5].repeat(1, 37, 1), ehs[1:, 40:].repeat(1, 5, 1)])  # repeated tokens share their weight: 185 of each
    ref = O.unet3d_forward(sd, cfg, sample, 601, short, pose, banks, do_cfg=True)
    assert T.nrmse(got, ref) < T.TOL


def _device_inputs(eng, sample, pose):
    b, _, f, hh, ww = sample.shape
    x = torch.zeros(b * f, hh, ww, 32, dtype=BF16, device="cuda")
    ops.pack_ncfhw(eng.lib, eng.stream, sample.cuda().contiguous(), x)
    cond = torch.zeros(b * f, hh, ww, 320, dtype=BF16, device="cuda")
    ops.pack_ncfhw(eng.lib, eng.stream, pose.cuda().contiguous(), cond)
    return x, torch.full((b,), 601.0, device="cuda"), cond


@pytest.mark.parametrize("tokens", [77, 1100])
def test_a_recorded_forward_reads_new_states(tokens):
    """recorded without an eager pass before it (1100 tokens: scratch that differs by level), replayed on new inputs and states with
    eager forwards of another executor and synchronisations between: each replay is the eager result, bit for bit"""
    from humanvid_amd.pipeline import StepRecorder

    cfg, sd, g, sample, ehs, pose, banks = _problem(tokens, 32)
    net, other = T.build_native(cfg, sd), T.build_native(cfg, sd)
    eng, eager = net.engine(), other.engine()

    def states(seed):
        gs = torch.Generator().manual_seed(seed)
        mask = torch.rand(2, tokens, generator=gs) < 0.7
        e = torch.randn(2, tokens, 768, generator=gs)
        for x in (eng, eager):
            x.set_encoder_hidden_states(e.cuda(), mask.cuda())

    for x in (eng, eager):
        x.set_reference_banks({k: v.cuda() for k, v in banks.items()}, do_cfg=True)
    states(1)
    x, t, cond = _device_inputs(eng, sample, pose)
    rec = StepRecorder(eng.lib)
    rec.begin()
    try:
        y = eng.forward_nhwc(x, t, cond, B=2, F=sample.shape[2])
    finally:
        rec.end()
    try:
        first = None
        for i in range(4):
            states(10 + i)
            x[..., :4].copy_(torch.randn(x[..., :4].shape, generator=g))
            rec.replay()
            torch.cuda.synchronize()
            got = y.clone()
            want = eager.forward_nhwc(x, t, cond, B=2, F=sample.shape[2])
            torch.cuda.synchronize()
            assert torch.equal(got, want) and bool(torch.isfinite(got).all())
            assert first is None or not torch.equal(got, first)
            first = got
    finally:
        rec.destroy()


def test_executors_of_the_halves():
    """each half by itself, made before the states are set: the rows of the whole batch (other tile selections: to rounding)"""
    cfg, sd, g, sample, ehs, pose, banks = _problem(77, 33)
    eng = T.build_native(cfg, sd).engine()
    eng.set_reference_banks({k: v.cuda() for k, v in banks.items()}, do_cfg=True)
    eng.set_encoder_hidden_states(torch.randn(2, 77, 768, generator=g).cuda())
    halves = [eng.clone_for_half(i) for i in (0, 1)]
    mask = torch.rand(2, 77, generator=g) < 0.5
    mask[:, 0] = True
    eng.set_encoder_hidden_states(ehs.cuda(), mask.cuda())
    x, t, cond = _device_inputs(eng, sample, pose)
    f = sample.shape[2]
    want = eng.forward_nhwc(x, t, cond, B=2, F=f).clone()
    for i, e in enumerate(halves):
        got = e.forward_nhwc(x[i * f:(i + 1) * f].contiguous(), t[:1], cond[i * f:(i + 1) * f].contiguous(), B=1, F=f)
        torch.cuda.synchronize()
        assert T.nrmse(got, want[i * f:(i + 1) * f]) < 1e-2, i


def test_product_in_ranges_under_graph_replays(cx):  # noqa: F811
    """quantise and multiply through one scratch, captured once and replayed on new data, with eager runs of other data between"""
    t, other = ec.ranges_tensors(cx, 1), ec.ranges_tensors(cx, 2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ec.ranges_run(cx.lib, s.cuda_stream, t)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ec.ranges_run(cx.lib, torch.cuda.current_stream().cuda_stream, t)
    for _ in range(4):
        t["x"].normal_()
        t["work"].fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        got = t["y"].clone(), t["y32"].clone()
        ec.ranges_run(cx.lib, cx.stream, other)
        for n in ("y", "y32"):
            t[n].zero_()
        t["work"].fill_(float("nan"))
        ec.ranges_run(cx.lib, cx.stream, t)
        torch.cuda.synchronize()
        assert torch.equal(got[0], t["y"]) and torch.equal(got[1], t["y32"]) and bool((t["y32"] != 0).any())


def test_products_in_ranges_on_two_streams(cx):  # noqa: F811
    """two runs at the same time, each with its own scratch, give what each gives alone"""
    both = [ec.ranges_tensors(cx, seed) for seed in (3, 4)]
    want = []
    for t in both:
        ec.ranges_run(cx.lib, cx.stream, t)
        torch.cuda.synchronize()
        want.append((t["y"].clone(), t["y32"].clone()))
        t["y"].zero_()
        t["y32"].zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for s, t in zip(streams, both):
            ec.ranges_run(cx.lib, s.cuda_stream, t)
    torch.cuda.synchronize()
    for t, w in zip(both, want):
        assert torch.equal(t["y"], w[0]) and torch.equal(t["y32"], w[1])


def test_command_list_of_a_product_in_ranges(cx):  # noqa: F811
    ec.case_ranges_command_list(cx)
