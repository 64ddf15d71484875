"""The scratch of attention over a cache in 4 bits, asked of the library: what is seen bounds it, and 1 GB does (or one key head of one sequence)."""
import ctypes

import pytest

from autogptq.tvm_b200 import _lib


def scratch(batch, heads, kv_heads, tokens, max_seq, hd=128, group=32, window=0, sinks=0):
    c = _lib.Cache4(dtype=0, batch=batch, kv_heads=kv_heads, max_seq=max_seq, hd=hd, group=group)
    a = _lib.AttnCacheArgs(cache=c, tokens=tokens, heads=heads, window=window, sinks=sinks, scale=1.0)
    return _lib.lib.b200gptq_attn_cache_workspace_bytes(ctypes.byref(a))


@pytest.mark.parametrize("batch,heads,kv_heads,tokens,max_seq", [
    (16, 32, 8, 16, 131072), (64, 32, 8, 16, 32768), (16, 32, 8, 64, 131072), (1, 32, 8, 512, 131072), (2, 72, 72, 512, 4224), (16, 64, 8, 4, 131072),
    (256, 32, 32, 64, 8192), (1, 1, 1, 4096, 1 << 20), (3, 40, 2, 700, 100003)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (256, 0), (4096, 4), (100000, 16)])
def test_scratch_is_bounded(batch, heads, kv_heads, tokens, max_seq, window, sinks):
    """What a query may see: all of the cache, or the window of all tokens and the sinks."""
    seen = min(max_seq, window + sinks + tokens - 1) if window else max_seq
    rows = 4 * 128 * seen                         # keys and values of one key head of one sequence
    bytes_ = scratch(batch, heads, kv_heads, tokens, max_seq, window=window, sinks=sinks)
    assert 0 <= bytes_ <= max(10 ** 9, rows) + 16 * batch
    assert bytes_ <= batch * kv_heads * rows + 16 * batch or bytes_ < 1 << 26      # (sums of the rows kernel: two for each of eight warps per SM, 32 rows of 130 numbers)


def test_a_window_takes_what_it_sees():
    """Sixteen texts in caches of 131072 rows, of which a window of 256 and 64 tokens see 319."""
    assert scratch(16, 32, 8, 64, 131072, window=256) == 16 * 8 * 319 * 128 * 4 + 16 * 8
    assert scratch(16, 32, 8, 64, 319, window=256) == 16 * 8 * 319 * 128 * 4
