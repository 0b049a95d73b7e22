"""What an engine with an 8-bit cache says of itself, and what the static deployment contracts make of it."""
import json

import pytest
import torch

from sdcguard_b200.evidence import config, operator_setup
from sdcguard_b200.ops import kv8
from sdcguard_b200.utils import stack


class _Engine:
    def __init__(self, cache):
        self.cache, self.max_model_len, self.sample_every, self.cuda_graph = cache, 512, 64, True


def test_stack_identity_names_the_caches_type():
    bf16 = torch.zeros(2, 4, 2, 2, 16, 128, dtype=torch.bfloat16)
    assert stack.collect(engine=_Engine(bf16))["kv_cache_dtype"] == "bfloat16"
    d = stack.collect(engine=_Engine(kv8.KV8Cache.empty(4, 2, 2, "cpu")))
    assert d["kv_cache_dtype"] == "float8_e4m3fn"
    assert d["fingerprint"] != stack.collect(engine=_Engine(bf16))["fingerprint"]


def test_page_bytes_by_the_cache_type():
    model = {"layers": 28, "kv_heads": 8, "head_dim": 128}
    assert config.kv_page_bytes(model, 16) == config.kv_page_bytes(model, 16, "bf16") == 28 * 2 * 8 * 16 * 128 * 2
    assert config.kv_page_bytes(model, 16, "fp8") == 28 * kv8.page_bytes(8)
    assert config.kv_page_bytes(model, 16, "int8") is None and config.kv_page_bytes(model, 16, ["fp8"]) is None


def _deployment(tmp_path, pages, lines, **over):
    d = json.loads(json.dumps(operator_setup.TEMPLATE))
    del d["workers"][1:]
    w = d["workers"][0]
    w.update(version="0.1.0", build="abc", kv_pages=pages, **over)
    (tmp_path / w["startup_log"]).write_text(f"sdcguard_b200 engine: kv_pages={pages} page_tokens=16{lines}\n")
    p = tmp_path / "d.json"
    p.write_text(json.dumps(d))
    doc, prov = config.load_deployment(str(p))
    return {r["id"]: r for r in config.assess(doc, prov)["workers"][0]["rules"]}


def test_capacity_counts_the_pages_of_the_declared_cache(tmp_path):
    """70000 pages: 128 GB in bf16, 64 GB in 8 bits, of 0.9 x 120 GB."""
    for kind, verdict in ((None, "violated"), ("bf16", "violated"), ("fp8", "satisfied"), ("int4", "unknown")):
        over = {} if kind is None else {"kv_cache": kind}
        rules = _deployment(tmp_path, 70000, "" if kind != "fp8" else " kv_cache=fp8", gpu_memory_gb=120, **over)
        assert rules["capacity.planned"]["verdict"] == verdict, kind
    pool = _deployment(tmp_path, 70000, " kv_cache=fp8", kv_cache="fp8")["capacity.planned"]["facts"]["pool_bytes"]
    assert pool == 70000 * 28 * kv8.page_bytes(8)


@pytest.mark.parametrize("declared,line,verdict", [
    (None, "", "satisfied"), ("bf16", "", "satisfied"), ("fp8", " kv_cache=fp8", "satisfied"),
    (None, " kv_cache=fp8", "violated"), ("fp8", "", "violated"), ("fp8", " kv_cache=bf16", "violated")])
def test_startup_line_has_the_declared_cache(tmp_path, declared, line, verdict):
    rules = _deployment(tmp_path, 70000, line, **({} if declared is None else {"kv_cache": declared}))
    assert rules["capacity.startup"]["verdict"] == verdict
