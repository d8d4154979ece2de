"""A cache that holds keys and values in 8 bits: storage, names and refusals (no GPU), and the plain statement itself."""
import dataclasses
import types

import numpy as np
import pytest
import torch

import plain_rows8 as R
from llmi_b200.cache.pages import CacheError
from llmi_b200.cache.storage import KVRequest, Rows8, SequenceCache
from llmi_b200.ops import kernels


@pytest.mark.parametrize("name,dtype", [("int8", torch.int8), ("float8_e4m3", torch.float8_e4m3fn)])
def test_storage_of_a_group_held_in_8_bits(name, dtype):
    cache = SequenceCache([(KVRequest(3, 64, held=name), 5)], [], 640, 1000, torch.bfloat16, "cpu")
    g = cache.kv_groups[0]
    assert g.k.dtype == g.v.dtype == dtype and g.k.shape == g.v.shape == (5, 10, 3, 64, 64)
    assert g.k_scale.shape == g.v_scale.shape == (5, 10, 3, 64) and g.k_scale.dtype == torch.float32
    k, v = g.rows8(2)
    assert isinstance(k, Rows8) and k.codes.data_ptr() == g.k[2].data_ptr() and v.scales.data_ptr() == g.v_scale[2].data_ptr()
    assert k.codes.is_contiguous() and k.scales.is_contiguous()
    assert cache.bytes_per_token() == 5 * 2 * 3 * (64 + 4)
    plain = SequenceCache([(KVRequest(3, 64), 5)], [], 640, 1000, torch.bfloat16, "cpu")
    assert plain.kv_groups[0].k_scale is None and plain.bytes_per_token() == 5 * 2 * 3 * 64 * 2


def test_an_unknown_type_is_refused():
    with pytest.raises(CacheError, match="int4"):
        SequenceCache([(KVRequest(3, 64, held="int4"), 1)], [], 64, 100, torch.bfloat16, "cpu")


def test_requests_with_and_without_8_bits_do_not_share_a_group():
    assert KVRequest(3, 64, held="int8") != KVRequest(3, 64)
    assert dataclasses.replace(KVRequest(3, 64, 7), held="int8") == KVRequest(3, 64, 7, held="int8")


def test_which_mixers_read_such_a_cache():
    from llmi_b200.engine.model import Model
    from llmi_b200.parts.attention import DiffAttention, GQAttention
    assert isinstance(GQAttention.holds_8bit, property) and not hasattr(DiffAttention, "holds_8bit")

    def model(**mixer):
        m = Model.__new__(Model)
        m.spec = types.SimpleNamespace(schedule=[types.SimpleNamespace(layer=0, cache_of=None)])
        m.layers = [types.SimpleNamespace(mixer=types.SimpleNamespace(kind="somekind", **mixer), parts={})]
        return m
    with pytest.raises(CacheError, match="somekind.*8 bits"):
        model(cache_request=lambda: KVRequest(2, 64)).new_cache(64, kv_type="int8")
    with pytest.raises(CacheError, match="no mixer of this model"):
        model(cache_request=lambda: None).new_cache(64, kv_type="int8")
    with pytest.raises(CacheError, match="bfloat16"):
        model(cache_request=lambda: KVRequest(2, 64), holds_8bit=True).new_cache(64, kv_type="bfloat16")
    assert model(cache_request=lambda: KVRequest(2, 64), holds_8bit=True)._mixer_request(0, "float8_e4m3") == KVRequest(2, 64, held="float8_e4m3")


def test_generate_refuses_a_type_beside_a_cache():
    from llmi_b200 import generate
    model = types.SimpleNamespace(spec=types.SimpleNamespace(stop_ids=()))
    with pytest.raises(ValueError, match="kv_type"):
        generate(model, [[1]], cache=object(), kv_type="int8")


def test_command_line():
    from llmi_b200.cli.generate import UsageError, parse_args
    assert parse_args(["dir", "--kv-type", "int8"])["kv_type"] == "int8" and parse_args(["dir"])["kv_type"] is None
    with pytest.raises(UsageError, match="kv-type"):
        parse_args(["dir", "--kv-type", "int4"])


def test_kernels_refuse_tensors_that_are_not_on_a_gpu():
    rows = Rows8(torch.zeros(1, 2, 64, 64, dtype=torch.int8), torch.zeros(1, 2, 64))
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(kernels.KernelError, match="CUDA"):
        kernels.rope_store8(torch.zeros(1, 8 * 64), torch.zeros(1, 4 * 64), None, 0, i, i, i.view(1, 1), rows, rows, 4, 2, 64)
    ctx = types.SimpleNamespace(tok_seq=i, tok_pos=i, seq_q_start=i, seq_kv_len=i, max_q_len=1)
    with pytest.raises(kernels.KernelError, match="CUDA"):
        kernels.attention8(torch.zeros(1, 4 * 64), torch.zeros(1, 4 * 64), rows, rows, ctx, i.view(1, 1), 4, 2, 64, 1.0)


def test_plain_e4m3_is_the_type_s_rounding():
    y = np.concatenate([np.random.default_rng(0).normal(size=4000) * 10.0 ** np.random.default_rng(1).uniform(-5, 2.5, 4000),
                        [0.0, 448.0, -448.0, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, 17.0, 19.0]]).astype(np.float32)
    ref = torch.from_numpy(np.clip(y, -448, 448)).to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(R.nearest_e4m3(y), ref)


@pytest.mark.parametrize("kind", ["int8", "float8_e4m3"])
def test_plain_rows(kind):
    x = np.random.default_rng(2).normal(size=(7, 24)) * 10.0 ** np.arange(-3, 4)[:, None]
    x[1] = 0.0
    x[2] = 2.0 ** -101
    x[3, 5] = np.inf
    codes, scale = R.held(x, kind)
    assert np.abs(codes).max() == R.MOST[kind] and (codes[1:4] == 0).all() and scale[1] == scale[2] == 0 and np.isnan(scale[3])
    fine = [0, 4, 5, 6]
    assert (np.abs(codes[fine] * scale[fine, None] - x[fine]) <= R.half_step(codes[fine], scale[fine], kind) * (1 + 1e-9)).all()


def test_parts_of_a_prompt_block_stay_within_the_launch():
    """However a step is made up: at least one part, none of fewer than four pages, and no more blocks than a grid has."""
    from llmi_b200.ops.kernels import prompt8_parts
    rng = np.random.default_rng(5)
    cut = 0
    for _ in range(4000):
        S, G, D = int(2 ** rng.uniform(0, 13)), int(rng.integers(1, 65)), int(rng.choice([64, 128]))
        rows = S + int(2 ** rng.uniform(0, 18))
        P = int(2 ** rng.uniform(0, 14))
        blocks = (rows + 255 * S) // 256
        n = prompt8_parts(rows, G, D, S, P, int(rng.integers(1, rows + 1)), 148)
        assert 1 <= n <= max(1, min(16, P // 4))
        if n > 1:
            cut += 1
            assert blocks * n <= 65535 and blocks * 32 <= 65535
    assert cut > 400
    assert prompt8_parts(400, 8, 128, 1, 63, 100, 148) == 9                       # two blocks of rows a kv head: 144 blocks in a wave
    assert prompt8_parts(2048, 32, 64, 1, 32, 2048, 148) == 1                     # a whole prompt that fills the device
