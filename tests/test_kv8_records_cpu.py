"""What an engine with an 8-bit cache says of itself."""
import torch

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
