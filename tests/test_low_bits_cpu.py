"""The engine's options in few bits, as far as they go without a GPU: configuration, cache layout, refusals, command line."""
import json

import pytest
import torch

from nanoinfer_b200.config import EngineConfig
from nanoinfer_b200.cache.storage import CacheStorage
from nanoinfer_b200.parts.base import CacheNeed, Runtime
from nanoinfer_b200.weights.int4 import Int4Matrix


def test_engine_config_refuses_what_it_does_not_know():
    assert EngineConfig().cache_dtype == "auto" and EngineConfig().weight_format == "auto"
    EngineConfig(cache_dtype="int8", weight_format="int4", weight_group=128)
    for bad in (dict(cache_dtype="fp8"), dict(cache_dtype="bfloat16"), dict(weight_format="int8"), dict(weight_group=48), dict(weight_group=0)):
        with pytest.raises(ValueError):
            EngineConfig(**bad)


def test_pages_of_8_bits_and_their_scales():
    full, window = CacheNeed.keys_and_values_int8(2, 64), CacheNeed.keys_and_values_int8(2, 64, 24)
    s = CacheStorage([(full, None, None), (window, None, None), (full, None, None)], 5, 16, 2, torch.bfloat16, "cpu")
    assert s.entry_group == [0, 1, 0]
    for e in range(3):
        p = s.pages[e]
        assert p["k"].shape == p["v"].shape == (5, 2, 16, 64) and p["k"].dtype == torch.int8
        assert p["k_scale"].shape == p["v_scale"].shape == (5, 2, 1, 1) and p["k_scale"].dtype == torch.float32
    # 2 x 2 x 64 codes a token, 2 x 2 floats a page of 16
    assert s.bytes_per_token() == 3 * (256 + 1)
    assert CacheStorage([(CacheNeed.keys_and_values(2, 64), None, None)], 5, 16, 2, torch.bfloat16, "cpu").bytes_per_token() == 512


def test_runtime_weights_are_matrices_unless_a_group_is_given():
    t = torch.randn(16, 64)
    plain = Runtime(torch.device("cpu"), torch.bfloat16, None)
    assert torch.equal(plain.weight(t), t.to(torch.bfloat16))
    w = Runtime(torch.device("cpu"), torch.bfloat16, None, False, 32).weight(t)
    assert isinstance(w, Int4Matrix) and w.shape == (16, 64) and w.group == 32


def _toy(tmp_path, cfg, **kw):
    from nanoinfer_b200.engine import Engine
    from nanoinfer_b200.registry import config_from_json_dict
    from nanoinfer_b200.weights import write_random_model
    from torch_ops import TorchOps
    d = str(tmp_path / "m")
    write_random_model(config_from_json_dict(cfg), d, seed=3)
    return Engine(d, EngineConfig(dtype="float32", page_size=8, num_pages=16, max_batch=2, device="cpu", **kw), ops=TorchOps())


def test_weight_bytes_of_a_model_in_4_bits(tmp_path):
    from tiny_configs import TINY_A
    plain, small = _toy(tmp_path, TINY_A), _toy(tmp_path, TINY_A, weight_format="int4", cache_dtype="int8")
    matrices = 2 * (64 * 128 + 64 * 64 + 3 * 64 * 128)
    assert plain.model.weight_bytes()[1] == small.model.weight_bytes()[1]
    n, b = small.model.weight_breakdown()["int4"]
    assert n == 8 and b == matrices // 2 + 2 * matrices // 64
    assert plain.model.weight_bytes()[0] - small.model.weight_bytes()[0] == 4 * matrices - b


def test_models_without_an_8_bit_form_are_refused(tmp_path):
    from nezalorn_util import CFG_A, DECAY_RANK, config_with_rank
    with pytest.raises(ValueError, match="8-bit"):
        _toy(tmp_path, config_with_rank(CFG_A, DECAY_RANK["A"]), cache_dtype="int8")


def test_a_matrix_whose_columns_no_group_divides_is_refused(tmp_path):
    from tiny_configs import TINY_W
    with pytest.raises(ValueError, match="multiple of 64"):
        _toy(tmp_path, TINY_W, weight_format="int4")


def test_commands_take_the_options(monkeypatch, tmp_path):
    import nanoinfer_b200.api as api
    from nanoinfer_b200.cli import generate, serve
    seen = []

    def fake(model_dir, **kw):
        seen.append(kw)
        raise KeyboardInterrupt

    monkeypatch.setattr(api, "load_model", fake)
    with open(tmp_path / "config.json", "w") as f:
        json.dump({}, f)
    for main, extra in ((generate.main, ["--prompt", "1"]), (serve.main, ["--prompt", "1"])):
        with pytest.raises(KeyboardInterrupt):
            main(["--model-dir", str(tmp_path), "--cache-dtype", "int8", "--weights", "int4", "--weight-group", "32"] + extra)
    assert all(k["cache_dtype"] == "int8" and k["weight_format"] == "int4" and k["weight_group"] == 32 for k in seen) and len(seen) == 2


def test_what_an_8_bit_cache_does_not_promise_is_said_where_it_is_promised():
    from nanoinfer_b200.api import Model
    from nanoinfer_b200.engine import scheduler
    from nanoinfer_b200.engine.engine import Engine
    for text in (Model.generate.__doc__, Engine.truncate.__doc__, scheduler.__doc__):
        assert "int8" in text or "8 bits" in text
