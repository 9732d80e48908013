"""The engine with a cache in 4 bits and matrices in 8 bits, on the CPU stand-in kernels: options, budget, whole runs."""
import types

import pytest
import torch

from leone_b200 import generate
from leone_b200.cache import packed
from leone_b200.engine.engine import Engine
from leone_b200.ops.int8 import quantize_matrix
from leone_b200.parts.base import PagedKV
from tests.emulated_ops import EmulatedOps
from tests.fewer_bits import quantize4, quantize8, values4
from tests.plain.model import PlainModel
from tests.tiny import make_folder


class FewerBitsOps(EmulatedOps):
    """Stand-ins for matrices in 8 bits and pages in 4 bits, from the 64-bit forms."""

    def prepare_matrix_int8(self, codes, scales, bias=None):
        self.calls.append("matrix8")
        return types.SimpleNamespace(codes=codes, scales=scales, bias=bias)

    def prepare_gate_up_int8(self, gc, gs, uc, us, gate_bias=None, up_bias=None):
        return self.prepare_matrix_int8(torch.cat([gc, uc]), torch.cat([gs, us]),
                                        None if gate_bias is None else torch.cat([gate_bias, up_bias]))

    def _product(self, x, w):
        if not hasattr(w, "codes"):
            return super()._product(x, w)
        a, s = quantize8(x.double())
        y = ((a @ w.codes.double().T) * s * w.scales.double()).float()
        return y if w.bias is None else y + w.bias

    def qk_norm_rope_write(self, ctx, qkv, n_q, n_kv, d, q_w, k_w, eps, table, rotary_dim, cache, pairing="half_split"):
        if cache is None or cache.bits is None:
            return super().qk_norm_rope_write(ctx, qkv, n_q, n_kv, d, q_w, k_w, eps, table, rotary_dim, cache, pairing=pairing)
        super().qk_norm_rope_write(ctx, qkv, n_q, n_kv, d, q_w, k_w, eps, table, rotary_dim, None, pairing=pairing)
        pos, seq = ctx.positions.long(), ctx.seq_of_token.long()
        page, slot = cache.block_table[seq, pos // cache.page_tokens].long(), pos % cache.page_tokens
        assert (page >= 0).all()
        rows = qkv.double().view(-1, n_q + 2 * n_kv, d)
        for pool, first, values in ((cache.k_pool, n_q, False), (cache.v_pool, n_q + n_kv, True)):
            codes, s, z = packed.unpack_pages(pool, d, values)
            new = quantize4(rows[:, first:first + n_kv])
            codes[page, :, slot] = new[0].to(torch.uint8)
            s[page, :, slot], z[page, :, slot] = new[1].to(torch.bfloat16), new[2].to(torch.bfloat16)
            pool.copy_(packed.pack_pages(codes, s, z, values))

    def attention(self, ctx, qkv, out, n_q, n_kv, d, scale, window, cache):
        if cache.bits is not None:
            k, v = (values4(*packed.unpack_pages(pool, d, values)).float() for pool, values in
                    ((cache.k_pool, False), (cache.v_pool, True)))
            cache = types.SimpleNamespace(k_pool=k, v_pool=v, block_table=cache.block_table, page_tokens=cache.page_tokens)
        super().attention(ctx, qkv, out, n_q, n_kv, d, scale, window, cache)


def _engine(folder, **kw):
    return Engine.from_folder(folder, **{**dict(dtype="float32", device="cpu", ops=FewerBitsOps(), page_tokens=16, max_tokens=512,
                                                max_requests=4, max_batch_tokens=64), **kw})


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    return make_folder(tmp_path_factory.mktemp("models"), "C")


def test_a_cache_in_4_bits_and_matrices_in_8_stay_near_the_plain_logits(folder):
    prompt = [(7 * i) % 200 for i in range(40)]
    want = PlainModel(folder).logits(prompt)
    full = want.std()
    for kw, near in (({}, 1e-4), ({"cache_bits": 4}, 0.2), ({"weight_bits": 8}, 0.2), ({"cache_bits": 4, "weight_bits": 8}, 0.3)):
        eng = _engine(folder, **kw)
        got = eng.step([("a", prompt[:25], list(range(25)))])
        got = torch.cat([got, eng.step([("a", prompt[25:], list(range(15)))])])
        off = float((got.double() - torch.as_tensor(want).double()).std() / float(full))
        assert (off < near) and (off > 1e-3 or not kw), (kw, off)
        assert ("matrix8" in eng.ops.calls) == ("weight_bits" in kw)
        assert eng.pools[0][0].dtype == (torch.uint8 if "cache_bits" in kw else torch.float32)


def test_pools_in_4_bits(folder):
    eng, full = _engine(folder, cache_bits=4), _engine(folder, dtype="bfloat16", ops=FewerBitsOps(torch.bfloat16))
    spec = eng.cache.groups[0].spec
    d = full.cache.groups[0].spec.head_dim
    assert spec.bits == 4 and spec.head_dim == packed.row_bytes(d) == spec.value_head_dim
    for pool in eng.pools[0]:
        assert pool.dtype == torch.uint8 and pool.shape[-1] == packed.row_bytes(d) and pool.shape[-2] == 16
    assert eng.memory_plan["cache"] * 2 * d == full.memory_plan["cache"] * packed.row_bytes(d)


def test_budget_of_matrices_in_8_bits(folder):
    eng, full = _engine(folder, weight_bits=8), _engine(folder)
    shapes = eng.model.matrices()
    assert len(shapes) == 4 * len(eng.model.blocks)
    saved = sum(r * c * 4 - (r * c + 4 * r) for r, c in shapes)
    assert eng.memory_plan["weights"] == full.memory_plan["weights"] - saved
    # never less than the upload of every tensor in its own type takes
    assert eng.memory_plan["required"] >= full.memory_plan["weights"]
    assert full.model.matrices() == []


def test_generate_takes_the_options(folder):
    ops = FewerBitsOps()
    eng = _engine(folder, ops=ops, cache_bits=4, weight_bits=8)
    out = generate(eng, [[5, 17, 3], [9] * 20], 4, use_graphs=False)
    assert [len(t) for t in out] == [4, 4]
    again = generate(_engine(folder, cache_bits=4, weight_bits=8), [[5, 17, 3], [9] * 20], 4, use_graphs=False, cache_bits=4, weight_bits=8)
    assert again == out
    with pytest.raises(ValueError, match="given engine"):
        generate(eng, [[5]], 1, cache_bits=4)


def test_refusals(folder):
    with pytest.raises(ValueError, match="4 bits"):
        _engine(folder, cache_bits=8)
    with pytest.raises(ValueError, match="8 bits"):
        _engine(folder, weight_bits=4)
    with pytest.raises(ValueError, match="multiple of 16"):
        _engine(folder, cache_bits=4, page_tokens=8)
    with pytest.raises(ValueError, match="4 bits"):
        PagedKV(2, 20, bits=4).resolved(torch.float32)
    with pytest.raises(ValueError, match="4 bits"):
        PagedKV(2, 64, value_head_dim=32, bits=4).resolved(torch.float32)
    with pytest.raises(ValueError, match="4 bits"):
        PagedKV(2, 64, bits=8).resolved(torch.float32)


def test_models_without_such_parts():
    # latent attention: its cache has no form in 4 bits
    from tests.sarizen_tiny import tiny_config
    from leone_b200.registry import spec_from_config
    spec = spec_from_config(tiny_config("R"))
    with pytest.raises(ValueError, match="cache_bits"):
        Engine(spec, random_seed=0, dtype="float32", device="cpu", ops=FewerBitsOps(), max_tokens=64, cache_bits=4)
    # rows of 72 elements are no whole number of 16 bytes
    with pytest.raises(ValueError, match="multiple of 16"):
        Engine(spec_from_config(tiny_config("Q")), random_seed=0, dtype="float32", device="cpu", ops=FewerBitsOps(), max_tokens=64,
               weight_bits=8)
    lightning = spec_from_config(tiny_config("P"))
    assert [s for s in Engine(lightning, random_seed=0, dtype="float32", device="cpu", ops=FewerBitsOps(), max_tokens=64,
                              weight_bits=8).model.matrices()] == [(96, 64), (64, 96)]


def test_quantize_matrix():
    g = torch.Generator().manual_seed(0)
    w = torch.randn((37, 48), generator=g)
    w[3] = 0
    w[5, 7] = float("inf")
    w[6, 0] = float("nan")
    codes, scales = quantize_matrix(w)
    want, s = quantize8(w.double())
    fine = [i for i in range(37) if i not in (5, 6)]
    assert torch.equal(codes[fine].double(), want[fine]) and torch.equal(scales[fine], s[fine, 0].float())
    assert scales[[5, 6]].isnan().all() and (codes[[5, 6]] == 0).all() and scales[3] == 0
    assert codes.abs().max() == 127
    with pytest.raises(ValueError, match="matrix"):
        quantize_matrix(w[0])


def test_command_line_takes_q4_and_int8():
    from leone_b200.cli import build_parser
    args = build_parser().parse_args(["generate", "-m", "x", "-t", "1", "-n", "2", "--kv", "q4", "--weights", "int8"])
    assert args.kv == "q4" and args.weights == "int8"
