"""GPU: MultiTensorAdamW in the framework's own adaptation step, beside optim.AdamW.

Both models enter every step with the same parameters, so the step's gradients are the same numbers; what may differ is the rounding
of the two kernels' updates: at most three of the parameter, and sixteen of a step no larger than 4 lr, for each step that the
moments have gone through (u = 2^-24)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from neat_amd import open_clip as oc, synth, train_TTA as T  # noqa: E402
from neat_amd.optim import AdamW, MultiTensorAdamW  # noqa: E402

DEV, U, LR = "cuda", 2.0 ** -24, 2e-4


def build(make, **kw):
    name = "neat-tiny"
    model = oc.create_model(name, device=DEV)
    model.load_state_dict(synth.synth_state_dict(name, 0))
    oc.freeze_parameters(model, False)
    params, _ = oc.collect_params(model, False)
    return model, params, make(params, lr=LR, weight_decay=1e-3, **kw)


def batches():
    cfg = synth.get_cfg("neat-tiny")
    t = cfg["text_cfg"]
    toks = [[x.to(DEV) for x in synth.synth_caption_sets(16, t["context_length"], t["vocab_size"], s)] for s in (1, 2, 3)]
    return toks, synth.synth_images(12, cfg["vision_cfg"]["image_size"], 7).to(DEV)


def test_steps_beside_the_flat_optimizer():
    (one, p1, o1), (two, p2, o2) = build(AdamW), build(MultiTensorAdamW)
    toks, images = batches()
    with torch.no_grad():
        gallery = one.encode_image(images, normalize=True)
    for k, tok in enumerate(toks, 1):
        for p, q in zip(p1, p2):
            q.data.copy_(p.data)
        was = [p.detach().clone() for p in p1]
        l1, i1, s1 = T.tta_step(one, o1, tok, gallery, 0.03, 0.07)
        l2, i2, s2 = T.tta_step(two, o2, tok, gallery, 0.03, 0.07)
        assert torch.equal(l1, l2) and torch.equal(i1, i2) and torch.equal(s1, s2)
        moved = 0.0
        for p, q, w in zip(p1, p2, was):
            assert ((p - q).abs() <= k * (3 * U * p.abs() + 16 * U * 4 * LR)).all()
            moved = max(moved, float((p - w).abs().max()))
        assert moved > 0.1 * LR
    assert o2._step_counts() == [3] * len(p2)


def test_steps_with_moments_in_8_bits_stay_finite_and_repeat():
    runs = []
    for _ in range(2):
        model, params, opt = build(MultiTensorAdamW, state_bits=8)
        toks, images = batches()
        with torch.no_grad():
            gallery = model.encode_image(images, normalize=True)
        runs.append([T.tta_step(model, opt, tok, gallery, 0.03, 0.07)[0] for tok in toks] + [p.detach().clone() for p in params])
    assert all(torch.equal(a, b) and torch.isfinite(a).all() for a, b in zip(*runs))
