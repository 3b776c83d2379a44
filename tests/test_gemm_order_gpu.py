"""The forward pass gives the same bits in every one of many steps, with the frozen tower's products beside the branch's kernels on the card: a wave of a product that is held up
in front of its loop must not find the ring's next tiles in the place of the one it reads."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_forward_same_bits_in_many_steps(gpu_lib):
    from dist_amd import synth
    from dist_amd.engine import Engine, config_from_geometry
    g = synth.geometry("b16_8+16f")
    eng = Engine(config_from_geometry(g, 32, torch.bfloat16))
    eng.load_state_dict(synth.state_dict(g))
    video = torch.from_numpy(synth.video(g, 32)).cuda()
    text = torch.from_numpy(synth.text_features(g)).cuda()
    target = torch.from_numpy(synth.soft_target(g, 32)[0]).cuda()
    first, feats = None, None
    for step in range(300):
        _, logits = eng.forward_backward(video, text, target)
        if first is None:
            first, feats = logits.clone(), eng.debug("feat.11").clone()
        elif not torch.equal(logits, first):
            rows = (eng.debug("feat.11") != feats).any(1).nonzero().flatten()
            raise AssertionError(f"step {step}: clips {(logits != first).any(1).nonzero().flatten().tolist()}, rows of the tower's output {rows[:8].tolist()}")
