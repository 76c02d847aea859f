"""TPDiTModulatedBlockINT8 over ranks, on the CPU: where its parameters are made, and a block of
two ranks (gloo) against one rank.  The INT8 kernels are replaced by the oracle-backed stand-in,
the operators around them by plain torch below."""
import os
import traceback
from pathlib import Path

import numpy as np
import pytest
import torch
import torch.multiprocessing as mp

import tp_worker
from test_tp_gloo import _port


# --------------------------------------------------------------------------------------
# devices
# --------------------------------------------------------------------------------------
@pytest.mark.parametrize("rank,world,device,want", [(0, 1, None, "cuda:0"), (1, 2, None, "cuda:1"),
                                                    (1, 2, "cuda:0", "cuda:0"), (1, 2, "cpu", "cpu")])
def test_every_parameter_is_made_on_one_device(monkeypatch, rank, world, device, want):
    """Without a device a rank's parameters lie on the GPU of its number, all of them."""
    from h3tp import tp_dit
    from h3tp.rms_rope import RotaryAxes
    made = []
    empty, ones = torch.empty, torch.ones

    def recorded(make):
        def on_meta(*a, device=None, **kw):
            made.append(torch.device(device))
            return make(*a, device="meta", **kw)
        return on_meta

    monkeypatch.setattr(torch, "empty", recorded(empty))
    monkeypatch.setattr(torch, "ones", recorded(ones))
    tp_dit.TPDiTModulatedBlockINT8(512, 512, 8, RotaryAxes(64, (64,)), 64, rank=rank, world_size=world,
                                   device=device)
    made = [d for d in made if d.type != "meta"]  # torch's own calls below the recorded ones
    assert set(made) == {torch.device(want)} and len(made) == 3 + 4 * 2 + 6


# --------------------------------------------------------------------------------------
# two ranks
# --------------------------------------------------------------------------------------
def _norm(v, spec):
    if spec is None:
        return v
    return v * torch.rsqrt((v * v).mean(1, keepdim=True) + spec.eps) * spec.weight


def _residual_norm(x, branch=None, gate=None, labels=None, *, post=None, pre=None, shift=None, scale=None,
                   quantize=False):
    v = x.float()
    if branch is not None:
        v = v + gate * _norm(branch.float(), post)
        x.copy_(v)
    if pre is None:
        return x, None, None
    h = _norm(v, pre) * (1 + scale) + shift
    if not quantize:
        return x, h.to(x.dtype), None
    h4 = torch.ones(4, 4) - 2 * torch.eye(4).flip(1)
    h16 = torch.kron(h4, h4)
    h = (h.unflatten(1, (-1, 256)) @ (torch.kron(h16, h16) / 16)).flatten(1)
    step = (h.abs().amax(1, keepdim=True) * (1 / 127)).clamp(min=1e-30)
    return x, torch.round(h / step).clamp(-128, 127).to(torch.int8), step


def _qk_norm_rope(q, k, positions, plan, *, q_weight=None, k_weight=None, eps=1e-6, norm=True, out_q=None,
                  out_k=None):
    angle = positions.double()[:, list(plan.axis_of_pair)] * torch.tensor(plan.inv_freq, dtype=torch.float64)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    for t, w, out in ((q, q_weight, out_q), (k, k_weight, out_k)):
        v = t.float()
        v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps) * w
        a, b = v[..., 0::2], v[..., 1::2]
        out.copy_(torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2))
    return out_q, out_k


def _int4_linear(x, weight, scales, zeros=None, *, group=128, bias=None, out_dtype=None):
    code = torch.stack((weight & 15, weight >> 4), 2).flatten(1)[:, :x.shape[1]].float()
    return x.float() @ ((code - 8) * scales.repeat_interleave(group, 1)[:, :x.shape[1]]).T + bias


def _attention(q, k, v):
    s = torch.einsum("shd,thd->hst", q.float(), k.float()) / q.shape[-1] ** 0.5
    return torch.einsum("hst,thd->shd", s.softmax(-1), v.float()).half()


HIDDEN, FFN, HEADS, COND, ROWS = 512, 1024, 8, 64, 40


def block_case(rank, world, port, outdir):
    try:
        dist = tp_worker._init(rank, world, port)
        from h3tp import ops, swiglu_quant
        from h3tp.rms_rope import RotaryAxes
        from h3tp.tp_dit import TPDiTModulatedBlockINT8
        ops.residual_norm, ops.qk_norm_rope, ops.int4_linear = _residual_norm, _qk_norm_rope, _int4_linear
        swiglu_quant.supported = lambda *a: True  # the contract but the device check holds here
        axes = RotaryAxes(64, (16, 24, 24))
        block = TPDiTModulatedBlockINT8(HIDDEN, FFN, HEADS, axes, COND, rank, world, device="cpu", comm=dist,
                                        group=32)
        g = torch.Generator().manual_seed(3)
        inner = HEADS * 64
        for m, (n, k) in ((block.qkv_proj, (3 * inner, HIDDEN)), (block.out_proj, (HIDDEN, inner)),
                          (block.fc1, (2 * FFN, HIDDEN)), (block.fc2, (HIDDEN, FFN))):
            m.load_shard_from_full(torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8),
                                   torch.rand(n, 1, generator=g) * 2e-4 + 1e-4)
        block.modulation.load_from_full(torch.randn(6 * HIDDEN, COND, generator=g) * 0.05,
                                        torch.randn(6 * HIDDEN, generator=g) * 0.2)
        for w in (block.attn_norm, block.attn_post_norm, block.mlp_norm, block.mlp_post_norm, block.q_norm,
                  block.k_norm):
            w.data.copy_(1 + 0.1 * torch.randn(w.numel(), generator=g))
        x = torch.randn(ROWS, HIDDEN, generator=g).half()
        cond = torch.randn(1, COND, generator=g).half()
        pos = torch.randint(0, 50, (ROWS, 3), generator=g, dtype=torch.int32)
        before = x.clone()
        with torch.no_grad():
            out = block(x, cond, pos, _attention)
        assert out is x and torch.isfinite(x).all()
        np.save(os.path.join(outdir, f"r{rank}.npy"), (x.double() - before.double()).numpy())
        dist.barrier()
        dist.destroy_process_group()
    except Exception:
        Path(outdir, f"err{rank}.txt").write_text(traceback.format_exc())
        raise


def test_two_ranks_agree_with_one(tmp_path):
    """Each rank ends with the same rows.  Against one rank, the partial sums travel as scaled
    fp16 (2^-12 of a value) and move some of the next codes by one step: at most what quantising
    itself does to each of the four quantised activations, (4 / 127) / sqrt(12) = 0.9% of its
    norm (a step is 1/127 of the maximum, about 4 standard deviations).  Heads, columns or rows
    on the wrong rank give errors of the size of the result."""
    got = {}
    for world in (1, 2):
        out = tmp_path / str(world)
        out.mkdir()
        mp.spawn(block_case, args=(world, _port(), str(out)), nprocs=world, join=True)
        got[world] = [np.load(out / f"r{r}.npy") for r in range(world)]
    assert np.array_equal(got[2][0], got[2][1])
    one, two = got[1][0], got[2][0]
    assert np.linalg.norm(two - one) <= 4 * 0.009 * np.linalg.norm(one)


# --------------------------------------------------------------------------------------
# shapes and policies that the second half of a forward could not run
# --------------------------------------------------------------------------------------
@pytest.mark.parametrize("ffn,world,policy", [
    (640, 1, {}), (1280, 2, {}), (1023, 2, {}), (0, 1, {}), (1024, 1, {"fc2_quantizer": "native"}),
    (1024, 1, {"fc2_quantizer": "owned_fp32"}), (1024, 1, {"row_linear_backend": "native"}),
    (640, 1, {"fc1_swiglu_epilogue": False})])
def test_block_refuses_what_fc2_cannot_take(ffn, world, policy):
    """Refused when the block is made, not after a forward has changed the residual."""
    from h3tp.h3_operator_policy import H3OperatorPolicy
    from h3tp.rms_rope import RotaryAxes
    from h3tp.tp_dit import TPDiTModulatedBlockINT8
    policy = H3OperatorPolicy(**{"fc1_swiglu_epilogue": True, **policy})
    with pytest.raises(ValueError):
        TPDiTModulatedBlockINT8(512, ffn, 8, RotaryAxes(64, (64,)), 64, 0, world, device="cpu", policy=policy)


@pytest.mark.parametrize("ffn,world,policy", [
    (1024, 2, {}), (1280, 2, {"fc1_swiglu_epilogue": False}),
    (1024, 1, {"fc1_swiglu_epilogue": False, "fc2_quantizer": "native"})])
def test_block_takes_what_fc2_takes(ffn, world, policy):
    from h3tp.h3_operator_policy import H3OperatorPolicy
    from h3tp.rms_rope import RotaryAxes
    from h3tp.tp_dit import TPDiTModulatedBlockINT8
    policy = H3OperatorPolicy(**{"fc1_swiglu_epilogue": True, **policy})
    TPDiTModulatedBlockINT8(512, ffn, 8, RotaryAxes(64, (64,)), 64, 0, world, device="cpu", policy=policy)
