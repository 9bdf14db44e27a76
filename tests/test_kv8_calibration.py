"""Calibrations and servers over 8-bit KV caches: tables, keys and serving commands name the cache they are for."""

import json
import logging

import pytest
import torch

from eagle4_b200 import api, cli
from eagle4_b200.core import live_costs
from eagle4_b200.core.live_costs import CostKey, check_kv_form, key_dtype, read_key, write_key


def _key(kv, engine="eagle4_b200"):
    return CostKey(gpu="x", gpu_count=1, model="m", draft="", engine=engine, dtype=key_dtype(kv))


def test_the_serving_command_and_the_workers_carry_the_cache_form(capsys):
    args = ["calibrate", "--model", "tiny", "--dry-run"]
    assert cli.main(args) == 0
    assert "--kv-dtype" not in capsys.readouterr().out
    assert cli.main(args + ["--kv-dtype", "int8"]) == 0
    assert "--kv-dtype int8" in capsys.readouterr().out
    assert cli.main(args + ["--kv-dtype", "fp8", "--tp", "2"]) == 0
    worker, serve = capsys.readouterr().out.strip().splitlines()[-2:]
    assert "--kv-dtype fp8" in worker and "--kv-dtype fp8" in serve


def test_no_packaged_profile_of_an_8_bit_cache(capsys):
    assert cli.main(["calibrate", "--model", "tiny", "--dry-run", "--package", "--kv-dtype", "int8"]) == 1
    assert "--package" in capsys.readouterr().err


@pytest.mark.parametrize("kv", [None, "int8"])
def test_packaged_profiles_serve_16_bit_caches_only(kv, monkeypatch):
    asked = []
    monkeypatch.setattr(api, "_with_packaged_profile", lambda config, *a: asked.append(1) or config)
    api.LLM.synthetic("tiny", device="cpu", dtype=torch.float32, tree=api.TreeSpec(2, 2, 4), max_len=32, kv_dtype=kv,
                      config=json.dumps({"mode": "serve"}))
    assert asked == ([1] if kv is None else [])


def test_tables_of_another_cache_form_are_named(tmp_path, caplog):
    assert key_dtype() == key_dtype("bf16") == "bfloat16"
    for stored, engine, ours, same in (("bf16", "eagle4_b200", None, True), ("bf16", "eagle4_b200", "int8", False),
                                       ("int8", "eagle4_b200", "int8", True), ("fp8", "eagle4_b200", "int8", False),
                                       ("fp8", "eagle4_b200", "bf16", False), ("bf16", "vllm", "int8", True)):
        write_key(str(tmp_path), _key(stored, engine))
        assert read_key(str(tmp_path)).dtype == key_dtype(stored)
        caplog.clear()
        with caplog.at_level(logging.WARNING, logger=live_costs.__name__):
            assert check_kv_form(str(tmp_path), ours) is same
        assert bool(caplog.records) is not same
    assert check_kv_form(str(tmp_path / "none"), "int8")


def test_an_engine_over_tables_of_another_cache_form_warns(tmp_path, caplog):
    write_key(str(tmp_path), _key("bf16"))
    config = json.dumps({"mode": "serve", "data_path": str(tmp_path)})
    for kv, warns in (("int8", True), ("bf16", False)):
        caplog.clear()
        with caplog.at_level(logging.WARNING, logger=live_costs.__name__):
            api.LLM.synthetic("tiny", device="cpu", dtype=torch.float32, tree=api.TreeSpec(2, 2, 4), max_len=32, kv_dtype=kv,
                              config=config)
        assert any("KV cache" in r.message for r in caplog.records) is warns


@pytest.mark.gpu
def test_calibrate_over_an_8_bit_cache(tmp_path):
    out = tmp_path / "cal"
    assert cli.main(["calibrate", "--model", "tiny", "--output", str(out), "--batch-sizes", "1,2", "--context-step", "64",
                     "--context-stop", "256", "--repeats", "2", "--steps", "2", "--top-k", "2", "--draft-tokens", "4",
                     "--kv-dtype", "int8"]) == 0
    assert read_key(str(out)).dtype == "bfloat16+kv_int8" and (out / "cost" / "bs_1").is_dir()
    assert "--kv-dtype int8" in (out / "serve.sh").read_text()
