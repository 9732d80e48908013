"""What the append of keys and values hands its kernels for the norm's weights."""
import types

import pytest
import torch

from leone_b200.cache import packed
from leone_b200.ops.cuda import CudaOps, KernelError
from leone_b200.parts.base import PagedCacheView

D, N_KV = 64, 2


class Calls:
    """Entry points that keep their arguments."""

    def __init__(self):
        self.args = None

    def __getattr__(self, name):
        def entry(*args):
            self.args = args
            return 0
        return entry


def _ops():
    ops = CudaOps.__new__(CudaOps)
    ops._pinned_stream, ops.launches = 0, 0
    ops.core_calls = ops.__dict__["_packed_calls"] = Calls()
    return ops


def _append(ops, q_w, k_w, bits):
    ints = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    pools = [torch.zeros((3, N_KV, 16, packed.row_bytes(D) if bits else D), dtype=torch.uint8 if bits else torch.bfloat16) for _ in range(2)]
    ctx = types.SimpleNamespace(positions=ints(1), seq_of_token=ints(1), status=ints(4))
    qkv = torch.zeros((1, (3 + 2 * N_KV) * D), dtype=torch.bfloat16)
    ops.qk_norm_rope_write(ctx, qkv, 3, N_KV, D, q_w, k_w, 1e-6, None, 0, PagedCacheView(*pools, ints(1, 3), 16, bits=bits))
    return ops.core_calls.args[6:9]


@pytest.mark.parametrize("bits", [None, 4])
@pytest.mark.parametrize("dtype,code", [(torch.float32, 0), (torch.bfloat16, 1)])
def test_weights_are_read_in_their_own_type(bits, dtype, code):
    q_w, k_w = torch.ones((2, D), dtype=dtype).unbind(0)
    ops = _ops()
    assert _append(ops, None, None, bits)[:2] == (None, None)
    for q in (q_w, None):                                    # a norm of the keys alone too
        have = _append(ops, q, k_w, bits)
        assert have[0] is q and have[1] is k_w and have[2] == code


@pytest.mark.parametrize("bits", [None, 4])
def test_weights_that_do_not_fit_are_refused(bits):
    ops, good = _ops(), torch.ones(D)
    for q_w, k_w in ((good, None), (None, torch.ones(D // 2)), (good, torch.ones(2 * D)), (good, good.bfloat16()),
                     (good, torch.ones(2 * D)[::2]), (torch.ones(2 * D)[::2], good), (None, torch.ones(2 * D)[::2])):
        with pytest.raises(KernelError, match="norm weights"):
            _append(ops, q_w, k_w, bits)
