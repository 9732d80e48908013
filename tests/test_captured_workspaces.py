"""Workspaces of captured decode steps in fewer bits: one memory for all of an engine's steps, which the budget counts."""
import pytest
import torch

from leone_b200.cache import packed
from leone_b200.engine.engine import Engine
from tests.test_fewer_bits_engine import FewerBitsOps
from tests.tiny import make_folder, tiny_config


def test_the_budget_counts_a_step_and_captured_steps(tmp_path):
    """Codes, gates beside their ups and parts of a step's largest layer, and twice those of a decode step: on the stream that captures, and
    in the graphs' memory.  (The plain path counts a step's gates and ups already.)"""
    folder = make_folder(tmp_path, "D")
    config = tiny_config("D")

    def scratch(max_requests, **kw):
        return Engine.from_folder(folder, dtype="float32", device="cpu", ops=FewerBitsOps(), page_tokens=16, num_pages=40, max_requests=max_requests,
                                  max_batch_tokens=128, **kw).memory_plan["scratch"]

    widths = config.hidden_size + config.num_attention_heads * config.head_dim + config.hidden_size + config.intermediate_size + 4 * 4
    for requests, captured in ((4, 2 * 4), (500, 2 * 128)):
        assert scratch(requests, weight_bits=8) - scratch(requests) == (128 + captured) * widths + captured * 2 * config.intermediate_size * 4
        assert scratch(requests, cache_bits=4) - scratch(requests) == packed.attention_workspace(64)
    # three times the parts of 444 blocks of 16 rows (of up to 128 numbers, a maximum and a sum), or of 2,048 of 8 rows
    assert packed.attention_workspace(256) >= 3 * 4 * 2048 * 8 * 258 and packed.attention_workspace(128) >= 3 * 4 * 444 * 16 * 130


@pytest.mark.gpu
def test_captured_decode_steps_share_their_workspaces(tmp_path):
    """Steps of one to ten requests, captured one after another and replayed in any order: each right, and the memory of one."""
    folder = make_folder(tmp_path, "D")
    engines = [Engine.from_folder(folder, dtype="bfloat16", page_tokens=16, num_pages=200, max_requests=12, max_batch_tokens=1024, cache_bits=4,
                                  weight_bits=8) for _ in range(2)]
    prompts = {r: [(11 * i + r) % 490 for i in range(30 + 9 * r)] for r in range(10)}
    for engine in engines:
        engine.ops.force_decode4_splits = 33                 # their parts go through a workspace
        engine.step([(r, p, [0]) for r, p in prompts.items()])
    captured, eager = engines
    sizes = [*range(1, 11), 4, 1, 10, 2, 7, 3]
    held = None
    for i, size in enumerate(sizes):
        tokens = [(5 * i + r) % 490 for r in range(size)]
        have = captured.decode_logits(list(range(size)), tokens).clone()
        want = eager.step([(r, [t], [0]) for r, t in enumerate(tokens)])
        # the same kernels, but for the forms of their launches
        assert float((have - want).norm() / want.norm()) < 0.03
        torch.cuda.synchronize()
        if held is None:
            held = torch.cuda.memory_reserved()
    # (the allocator takes 2 MiB at a time for small tensors, and a pool of its own for a graph takes that at least)
    assert torch.cuda.memory_reserved() - held <= 6 << 20


@pytest.mark.gpu
def test_captured_steps_that_make_room_for_others(tmp_path):
    """Sizes that are captured, dropped and captured again beside others, whose graphs lie in the same memory."""
    folder = make_folder(tmp_path, "D")
    engines = [Engine.from_folder(folder, dtype="bfloat16", page_tokens=16, num_pages=100, max_requests=6, max_batch_tokens=512, cache_bits=4,
                                  weight_bits=8) for _ in range(2)]
    captured, eager = engines
    for most in (1, 2):
        captured.max_decode_graphs = most
        for engine in engines:
            engine.ops.force_decode4_splits = 33
            engine.step([((most, r), [(11 * i + r) % 490 for i in range(20 + 9 * r)], [0]) for r in range(5)])
        for i, size in enumerate((1, 2, 3, 4, 5, 2, 1, 5, 2, 2, 4, 1)):
            tokens = [(5 * i + r) % 490 for r in range(size)]
            have = captured.decode_logits([(most, r) for r in range(size)], tokens).clone()
            want = eager.step([((most, r), [t], [0]) for r, t in enumerate(tokens)])
            assert float((have - want).norm() / want.norm()) < 0.03
            assert len(captured._decode_graphs) <= most
        for engine in engines:
            for r in range(5):
                engine.close((most, r))
