"""SparseVoxel with sorted_lookup: the switch reaches every path that computes a
gradient of the embeddings, and equal batches give equal bits."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(__file__))
import voxfusion_golden_util as vg  # noqa: E402

from xrdslam_amd.slam.common.camera import Camera  # noqa: E402
from xrdslam_amd.slam.configs.input_config import (  # noqa: E402
    cadence, voxfusion_config)
from xrdslam_amd.slam.models.sparse_voxel import SparseVoxelConfig  # noqa: E402

DEV = 'cuda:0'
CAM = dict(fx=150., fy=150., cx=79.5, cy=59.5, width=160, height=120)


def algorithm(sorted_lookup, device):
    config = voxfusion_config()
    config.model.sorted_lookup = sorted_lookup
    return config.setup(camera=Camera(**CAM), device=device)


def test_the_switch_is_a_field_of_the_configuration():
    assert SparseVoxelConfig().sorted_lookup is False
    for on in (False, True):
        algo = algorithm(on, 'cpu')
        assert algo.model.sorted_lookup is on
        # mapping leaves the fixed launch sequence, tracking (no gradient of
        # the embeddings) does not
        assert algo._fused(True) is not on and algo._fused(False)
        algo.use_graphs = True
        if on:
            assert not algo._graphs_ok(None, True)
            assert algo.map_slot_key(10, [None], False) is None


def test_a_batch_without_hits_is_no_end(monkeypatch):
    """(rendering answers None then; the fused iteration goes on)"""
    algo = algorithm(True, 'cpu')
    monkeypatch.setattr(type(algo), 'get_model_input', lambda *_: {})
    monkeypatch.setattr(type(algo.model), 'forward', lambda *_: None)
    loss = algo.get_loss([None], True, 0, 1)
    loss.backward()
    assert float(loss) == 0.0
    assert all(p.grad is None for p in algo.model.parameters())


def forbid_fused(monkeypatch):
    """the kernels that add the embeddings' gradient by atomics"""
    from xrdslam_amd.engine import vox

    def never(*_, **__):
        raise AssertionError('fused')
    monkeypatch.setattr(vox, 'points', never)
    monkeypatch.setattr(vox, 'render_loss', never)


@pytest.mark.gpu
@pytest.mark.parametrize('which', ['small', 'office0'])
def test_golden_through_the_sorted_lookup(which, monkeypatch):
    """the recorded model, losses and gradients, at the bound that every path
    through this model is held to"""
    g = vg.Golden(vg.GOLDEN if which == 'small' else vg.GOLDEN_OFFICE0)
    model = vg.build_model(g, DEV)
    model.sorted_lookup = True
    forbid_fused(monkeypatch)
    exact, errs = vg.run(model, g, DEV, True)
    assert all(exact.values()), exact
    bad = {k: v for k, v in errs.items() if not v < 1e-4}
    assert not bad, bad


def room(sorted_lookup, n_frames=40):
    from xrdslam_amd.data.synthetic import SyntheticRoom
    from xrdslam_amd.slam.pipeline import SequentialSLAM
    torch.manual_seed(0)
    algo = algorithm(sorted_lookup, DEV)
    data = SyntheticRoom([[-3, 3], [-4, 2.5], [-2, 2.5]], H=120, W=160,
                         fx=150., fy=150., cx=79.5, cy=59.5, n_frames=n_frames,
                         device=DEV)
    cad = cadence['vox-fusion']
    return algo, SequentialSLAM(
        algo, data, map_every=cad.map_every, keyframe_every=cad.keyframe_every,
        pose_device=DEV, use_relative_pose=cad.use_relative_pose,
        init_pose_offset=cad.init_pose_offset)


@pytest.mark.gpu
def test_mapping_gradients_repeat(monkeypatch):
    algo, slam = room(True)
    algo.use_graphs = True
    slam.step(0)
    frame = algo.keyframe_graph[0]
    model = algo.model
    model.noise_fn = lambda shape, like: like.new_full(shape, 0.5)
    inp = algo.get_model_input([frame], True)
    inp = {k: v.detach() if torch.is_tensor(v) else v for k, v in inp.items()}
    algo.get_model_input = lambda *_: dict(inp)
    forbid_fused(monkeypatch)
    seen = []
    for _ in range(4):
        model.zero_grad(set_to_none=True)
        algo.get_loss([frame], True, 0, 1).backward()
        seen.append(model.embeddings.grad.clone())
        torch.empty(1 << 20, device=DEV).normal_()      # other work between
    assert seen[0].abs().max() > 0
    assert all(torch.equal(s, seen[0]) for s in seen)


@pytest.mark.gpu
def test_the_loop_runs():
    """tracking through its captured graph, mapping through the lookup"""
    algo, slam = room(True)
    algo.use_graphs = True
    for k in range(7):
        slam.step(k)
    assert algo._track_slot['graph'] is not None
    assert not getattr(algo, '_map_slots', {})
    assert torch.isfinite(algo.model.embeddings).all()
    rgb, depth = algo.render_img(algo.get_estimate_c2w_list()[5].to(DEV))
    assert (depth > 0).mean() > 0.5
