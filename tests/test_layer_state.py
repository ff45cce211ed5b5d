"""The cache of a causal layer when one of its calls is refused (no GPU: the operators are stand-ins)."""
import pytest
import torch

import brodiffusion_b200 as bd
from brodiffusion_b200 import layer as LY

CALLS = ["add_rmsnorm_fwd", "linear_act_fwd", "rmsnorm_rope", "sdpa_window_fwd"]


@pytest.mark.parametrize("refused", range(9))
def test_a_refused_call_leaves_the_cache_as_it_was(monkeypatch, refused):
    D, nh, nkv, hd, F, B = 64, 2, 1, 32, 128, 3
    w = dict(norm1=torch.ones(D), norm2=torch.ones(D), wqkv=torch.ones((nh + 2 * nkv) * hd, D), wo=torch.ones(D, nh * hd),
             w_up=torch.ones(F, D), w_down=torch.ones(D, F))
    L = LY.CausalLayer({n: t.bfloat16() for n, t in w.items()}, nh, nkv, hd, window=4)
    cache = LY.KvCache(B, 16, nkv, hd, torch.bfloat16, device="cpu")
    cache.filled, lengths = [5, 0, 9], cache.lengths
    lengths.copy_(torch.tensor(cache.filled))
    made = []

    def stand_in(name):
        def call(*args, **kw):
            made.append(name)
            if name == "sdpa_window_fwd":
                assert kw["kv_len"].tolist() == [7, 2, 11]            # the new rows are seen
            if len(made) == refused + 1:
                raise bd.BdattnError("refused")
        return call
    for name in CALLS:
        monkeypatch.setattr(bd, name, stand_in(name))
    cos = torch.zeros(16, hd // 2)
    x = torch.zeros(B, 2, D, dtype=torch.bfloat16)
    with pytest.raises(bd.BdattnError, match="refused"):
        L.forward(x, cache, cos, cos)
    assert cache.filled == [5, 0, 9] and cache.lengths is lengths and lengths.tolist() == [5, 0, 9]
    made.append("no more")
    L.forward(x, cache, cos, cos)
    assert cache.filled == [7, 2, 11] and cache.lengths is lengths and lengths.tolist() == [7, 2, 11]
