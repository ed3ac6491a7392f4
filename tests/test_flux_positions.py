"""The positions of each image's own as a run's conditioning holds them: any type, no value changed."""

from __future__ import annotations

import pytest
import torch

from selas_amd import flux as F

from .conftest import seeded

F16, F32, F64, I16, I32, I64 = torch.float16, torch.float32, torch.float64, torch.int16, torch.int32, torch.int64


def prepared(txt, img, b=2):
    return F._positions_of_each(txt, img, b, torch.device("cpu"))


@pytest.mark.parametrize("txt_t,img_t,want", [(F32, I64, F32), (F32, I32, F32), (F16, I64, F32), (F64, F32, F32)])
def test_fractions_of_the_text_stay(txt_t, img_t, want):
    txt = torch.tensor([[0.5, 0.0, -2.25], [1.0, 3.5, 0.0]], dtype=txt_t)
    img = torch.arange(12).view(2, 2, 3).to(img_t)
    ids = prepared(txt, img)
    assert ids.dtype == want and ids.shape == (2, 4, 3)
    assert torch.equal(ids[:, :2].double(), txt.double().expand(2, 2, 3)) and torch.equal(ids[:, 2:].double(), img.double())


@pytest.mark.parametrize("txt_t,img_t,want", [(F32, I64, I64), (F32, I32, I32), (I64, I32, I32), (I64, F32, F32), (F32, I16, F32),
                                              (F32, F16, F32), (F32, torch.bfloat16, F32), (F32, F64, F32), (F64, F64, F32)])
@pytest.mark.parametrize("shared", [False, True])
def test_whole_numbers_of_every_type(txt_t, img_t, want, shared):
    txt, img = torch.zeros(5, 3).to(txt_t), torch.arange(0, 96, 4).view(2, 4, 3).to(img_t)
    img = img[:1] if shared else img
    ids = prepared(txt, img)
    assert ids.dtype == want and torch.equal(ids.double(), torch.cat((txt.expand(2, 5, 3).double(), img.expand(2, 4, 3).double()), 1))


def test_far_whole_numbers_stay_exact():
    img = torch.tensor([[[0, 1 << 40, (1 << 24) + 1]]])
    assert torch.equal(prepared(torch.zeros(1, 3), img, 1)[0, 1], img[0, 0])


@pytest.mark.parametrize("txt,img", [(torch.zeros(1, 3), torch.full((2, 1, 3), 0.1, dtype=F64)),
                                     (torch.full((1, 3), 0.5), torch.full((2, 1, 3), (1 << 24) + 1))])
def test_values_that_no_type_holds_are_refused(txt, img):
    with pytest.raises(ValueError, match="float32 does not hold"):
        prepared(txt, img)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_positions_that_are_not_finite_are_no_whole_numbers(value):
    ids = prepared(torch.tensor([[0.0, value, 1.0]]), torch.ones(1, 2, 3, dtype=I64), 1)
    assert ids.dtype == F32 and torch.equal(ids[0, 0, 1].isnan(), torch.tensor(value != value))
    assert value != value or ids[0, 0, 1] == value


def test_a_batch_of_another_size_is_refused():
    with pytest.raises(ValueError, match="batch of 2"):
        prepared(torch.zeros(1, 3), torch.zeros(3, 1, 3))


@pytest.mark.gpu
def test_every_type_gives_one_result(dev):
    cfg = F.FluxConfig(hidden=256, heads=2, mlp_hidden=512, depth_double=1, depth_single=1, in_channels=64, context_dim=128,
                       vec_dim=64, axes_dim=(16, 56, 56))
    runner = F.FluxRunner(F.RandomFlux(cfg, dev, seed=3, quant="raw"))
    g = seeded(4)
    pooled, txt, lat = torch.randn(2, 64, generator=g), torch.randn(2, 3, 128, generator=g), torch.randn(2, 12, 64, generator=g)
    own = torch.stack((F.image_ids(3, 4), F.image_ids(4, 3) + 2.0))
    for text in (F.text_ids(3), F.text_ids(3) + 0.5):
        outs = []
        for dtype in (F32, I64, F16, F64, I32):
            cond = runner.prepare([1.0, 0.5], 3.5, pooled, txt, own.to(dtype), text)
            assert torch.equal(cond.ids[0, :3].cpu().double(), text.double())
            outs.append(runner.step(0, lat.to(dev), cond)[0])
        assert all(torch.equal(outs[0], o) for o in outs[1:])
