"""What a program may read of the MoE engine after read_state()."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_parameters_are_those_of_the_finished_step_after_read_state(dev):
    """The optimizer's stream is held up for some milliseconds: work queued on the current stream after read_state() comes behind it all the same."""
    from internevo_amd.config import ModelConfig, PathConfig, TrainConfig
    from internevo_amd.data import SyntheticLoader
    from internevo_amd.moe_engine import MoEEngine

    mc = ModelConfig(vocab_size=512, hidden_size=256, num_layers=2, num_attention_heads=2, num_kv_attention_heads=2, mlp_ratio=8 / 3, model_type="INTERNLM", num_experts=1)
    tc = TrainConfig(seq_len=256, micro_bsz=1, micro_num=2, total_steps=4, lr=1e-3, fixed_random_dataset_seqlen=True)
    eng = MoEEngine(PathConfig(mc, tc), dev, seed=5)
    before = eng.params.clone()
    batch, labels = next(iter(SyntheticLoader(256, 1, 2, True, 8)))
    eng.forward_backward(batch, labels)
    torch.cuda.synchronize()
    with torch.cuda.stream(eng.opt_stream):
        torch.cuda._sleep(50_000_000)
    eng.step()
    eng.read_state()
    after = eng.params.clone()
    torch.cuda.synchronize()
    assert torch.equal(after, eng.params) and not torch.equal(after, before)
