"""What DecodeBatch refuses on the host, before a kernel reads an address: metadata and
results of another type than the kernels take, as `torch.empty(..., dtype=config.dtype)` makes them
for a cache held in 8 bits."""

from types import SimpleNamespace

import pytest
import torch

from hisparse_b200 import CacheConfig, DecodeBatch, HotConfig

E4M3 = torch.float8_e4m3fn
SHAPE = (1, 4, 2, 32)


def cache_of(dtype):
    return SimpleNamespace(config=CacheConfig(gpu_pages=4, page_size=4, dtype=dtype, device="cpu"),
                           hot_config=HotConfig(8), compute=None, transfer=None,
                           device=torch.device("cpu"))


@pytest.mark.parametrize("cache,given", [(E4M3, E4M3), (E4M3, torch.float32),
                                         (E4M3, torch.float16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("which", [0, 1])
def test_metadata_of_another_type(cache, given, which):
    cache = cache_of(cache)
    bounds = [{r: torch.empty(SHAPE, dtype=cache.config.metadata_dtype) for r in range(2)}
              for _ in range(2)]
    bounds[which][1] = torch.empty(SHAPE, dtype=given)
    with pytest.raises(ValueError, match=f"must be {cache.config.metadata_dtype}"):
        DecodeBatch(cache, range(2), 1, *bounds, 2, 4)


@pytest.mark.parametrize("out", [
    torch.empty(2, 4, 32, dtype=E4M3), torch.empty(2, 4, 32, dtype=torch.float32),
    torch.empty(2, 4, 16, dtype=torch.bfloat16), torch.empty(2, 32, 4, dtype=torch.bfloat16).mT])
def test_results_of_another_kind(monkeypatch, out):
    batch = object.__new__(DecodeBatch)
    batch.config, batch.layers = cache_of(E4M3).config, [None]
    batch.batch, batch.q_heads, batch.device, batch.compute = 2, 4, torch.device("cpu"), "stream"
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *_: "stream")
    with pytest.raises(ValueError, match="out must be"):
        batch.layer(0, torch.empty(2, 4, 32, dtype=torch.bfloat16), out)
