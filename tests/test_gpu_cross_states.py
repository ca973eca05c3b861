"""UNet forwards with encoder states of several tokens on a real MI355X, against the oracle.

Tolerance: that of the one-token forwards (tests/test_gpu_unet.py: NRMSE <= 2e-2, bf16 storage against fp32); a masked token is the
same as an absent one."""
import pytest
import torch

import test_gpu_unet as T

O = T.O
pytestmark = pytest.mark.gpu


def _inputs(cfg, f, hh, ww, tokens, seed):
    g = torch.Generator().manual_seed(seed)
    sample = torch.randn(1, 4, f, hh, ww, generator=g).repeat(2, 1, 1, 1, 1)
    ehs = torch.randn(2, tokens, 768, generator=g)
    pose = (torch.randn(1, cfg["block_out_channels"][0], f, hh, ww, generator=g) * 0.5).repeat(2, 1, 1, 1, 1)
    return sample, ehs, pose


def test_unet3d_with_a_prompt():
    cfg = O.tiny_unet3d_cfg()
    sd = O.make_unet3d_weights(cfg, seed=0)
    net = T.build_native(cfg, sd)
    sample, ehs, pose = _inputs(cfg, 4, 8, 8, 77, 3)
    one = T.run_native(net, sample, 601, ehs[:, :1], pose, None, do_cfg=False)
    out = T.run_native(net, sample, 601, ehs, pose, None, do_cfg=False)
    ref = O.unet3d_forward(sd, cfg, sample, 601, ehs, pose, None, do_cfg=False)
    assert T.nrmse(out, ref) < T.TOL
    assert T.nrmse(out, one) > 1e-2  # the states matter
    # masked tokens are absent ones, whatever they hold
    mask = torch.rand(1, 77, generator=torch.Generator().manual_seed(5)) < 0.5
    mask[:, 0] = True
    spoiled = ehs.masked_fill(~mask[..., None], float("nan"))
    eng = net.engine()
    got = net(sample.cuda(), 601, spoiled.cuda(), pose_cond_fea=pose.cuda(), return_dict=False,
              encoder_attention_mask=mask.expand(2, -1).cuda())[0]
    ref = O.unet3d_forward(sd, cfg, sample, 601, ehs[:, mask[0]], pose, None, do_cfg=False)
    assert bool(torch.isfinite(got).all()) and T.nrmse(got, ref) < T.TOL
    # and one token again gives the bits it gave before
    again = T.run_native(net, sample, 601, ehs[:, :1], pose, None, do_cfg=False)
    assert torch.equal(again, one) and not eng.cross_kv


def test_unet3d_with_image_tokens_head_dim_160():
    cfg = O.tiny_unet3d_cfg(block_out_channels=(320, 1280))
    sd = O.make_unet3d_weights(cfg, seed=1)
    net = T.build_native(cfg, sd)
    sample, ehs, pose = _inputs(cfg, 2, 16, 8, 257, 4)
    out = T.run_native(net, sample, 32, ehs, pose, None, do_cfg=False)
    ref = O.unet3d_forward(sd, cfg, sample, 32, ehs, pose, None, do_cfg=False)
    assert T.nrmse(out, ref) < T.TOL


def test_reference_net_with_a_prompt():
    from humanvid_amd.reference_control import ReferenceAttentionControl
    from humanvid_amd.unet2d import UNet2DConditionModel

    cfg = O.tiny_unet3d_cfg()
    sd = O.make_reference_net_weights(cfg, seed=5)
    types = dict(down_block_types=("CrossAttnDownBlock2D", "DownBlock2D"), up_block_types=("UpBlock2D", "CrossAttnUpBlock2D"))
    net = UNet2DConditionModel(**{**{k: v for k, v in cfg.items() if k in ("block_out_channels", "layers_per_block", "cross_attention_dim")}, **types})
    net.load_state_dict(sd, strict=True)
    net = net.to("cuda")
    g = torch.Generator().manual_seed(7)
    lat, ehs = torch.randn(1, 4, 8, 8, generator=g), torch.randn(1, 20, 768, generator=g)
    writer = ReferenceAttentionControl(net, do_classifier_free_guidance=False, mode="write", batch_size=1, fusion_blocks="full")
    net(lat.cuda(), torch.zeros(()), ehs.cuda())
    want = O.reference_net_banks(sd, cfg, lat, ehs)
    blocks = {n.rsplit(".transformer_blocks.0", 1)[0]: m for n, m in net.named_modules() if hasattr(m, "bank") and len(getattr(m, "bank"))}
    assert set(blocks) == set(want)
    for n, m in blocks.items():
        assert T.nrmse(m.bank[0], want[n]) < T.TOL, n
    writer.clear()
