"""CPU: checks of the training-step operators' Python entries that need no GPU: counts past 32 bits, options of an optimiser's groups, models that
take no group norm."""
import random

import pytest
import torch

from openpcdet_amd import _lib, backbones_2d, focal, optim, unet


# ---- counts ----------------------------------------------------------------------------------------------------------------
def test_counts_past_32_bits():
    _lib.check_counts("op", 0, 1, 2 ** 31 - 1)
    for big in (2 ** 31, 2 ** 32 + 5):
        with pytest.raises(ValueError, match="op: a count of %d is past 32 bits" % big):
            _lib.check_counts("op", 3, big, 1)


# ---- the optimiser's options -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kw", [dict(steps=100), dict(steps=-1), dict(coefficients=(3.0, -2.0, 0.0)), dict(coefficients=(1.0, 2.0)), dict(eps=-1.0),
                                dict(eps=float("nan")), dict(momentum=-3.0), dict(momentum=1.0), dict(weight_decay=-1.0), dict(lr=-1.0)])
def test_muon_refuses_options_of_a_group(kw):
    w, v = (torch.nn.Parameter(torch.zeros(4, 4)) for _ in range(2))
    with pytest.raises(ValueError):
        optim.Muon([dict(params=[w], **kw)])
    with pytest.raises(ValueError):
        optim.Muon([w], **kw)
    opt = optim.Muon([w])
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=[v], **kw))
    assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=[v], lr=0.1, momentum=0.5))           # refused groups leave nothing behind
    assert [g["momentum"] for g in opt.param_groups] == [0.95, 0.5]


def test_muon_refuses_matrices_past_the_largest():
    for shape in ((2 ** 20 + 1, 1), (1, 2 ** 20 + 1), (2, 2 ** 10, 2 ** 10 + 1)):
        w = torch.nn.Parameter(torch.zeros(shape))
        w.grad = torch.zeros(shape)
        with pytest.raises(ValueError, match="1048576"):
            optim.Muon([w]).step()


# ---- NORM_GROUPS -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("make", [unet.UNetV2, focal.VoxelBackBone8xFocal, backbones_2d.PillarBackBone8x, backbones_2d.PillarRes18BackBone8x,
                                  backbones_2d.VoxelResBackBone8xVoxelNeXt2D])
def test_models_without_group_norm_say_so(make):
    """the key is of the voxel backbones: a model that has BatchNorm only must not take it for nothing"""
    with pytest.raises(ValueError, match="NORM_GROUPS"):
        make(model_cfg={"NORM_GROUPS": 4}, input_channels=5, grid_size=[64, 64, 40])


# ---- coefficients ----------------------------------------------------------------------------------------------------------
def test_accepted_polynomials_are_their_slope_near_zero():
    """the range that is followed starts at 1/64; below it, where more than 4096 equal singular values start, a + b y + c y^2 has to be a"""
    r, taken = random.Random(1), 0
    for _ in range(50000):
        a = r.uniform(-4, 4)
        b, c = a * r.uniform(-12, 12), a * r.uniform(-12, 12)
        if _lib.lib().pvx_orthogonalize_holds(1, a, b, c):
            taken += 1
            assert max(abs(b * y + c * y * y) for y in (2.0 ** -12, 2.0 ** -13)) <= 0.01 * abs(a)
    assert taken > 500
