"""Host side of the serving operators without a GPU: argument checks of the C
entries (no device work is queued for them) and the prompt plan."""

import ctypes

import numpy as np
import pytest

from xpu_playground_b200 import _lib

INVALID, UNSUPPORTED = _lib.XPU_ERR_INVALID, _lib.XPU_ERR_UNSUPPORTED


def cache(**change):
    fields = dict(k=64, v=64, tables=64, lens=64, refs=64, status=64, workspace=64, dtype=0, layers=2, pages=10, page_size=16,
                  kv_heads=2, head_dim=64, sequences=4, table_width=5) | change
    return ctypes.byref(_lib.KvCacheC(**fields))


def compact(**change):
    return _lib.load().xpu_kv_compact(cache(**change), None)


@pytest.mark.parametrize("change,status", [
    ({"k": None}, INVALID), ({"refs": None}, INVALID), ({"workspace": None}, INVALID), ({"v": 8}, INVALID),
    ({"dtype": 2}, INVALID), ({"layers": 0}, INVALID), ({"pages": 0}, INVALID), ({"sequences": 0}, INVALID),
    ({"page_size": 24}, UNSUPPORTED), ({"page_size": 256}, UNSUPPORTED), ({"head_dim": 96}, UNSUPPORTED),
    ({"sequences": 65537}, INVALID), ({"pages": 1 << 30}, INVALID), ({"table_width": 1 << 28}, INVALID),
])
def test_cache_refusals(change, status):
    assert compact(**change) == status
    assert "xpu_kv_compact" in _lib.last_error()


def test_null_cache_and_lists():
    L = _lib.load()
    assert L.xpu_kv_compact(None, None) == INVALID
    assert L.xpu_kv_extend(cache(), None, 64, 1, None) == INVALID
    assert L.xpu_kv_trim(cache(), 64, None, 1, None) == INVALID
    assert L.xpu_kv_fork(cache(), 64, 64, 1025, None) == INVALID
    assert L.xpu_kv_fork(cache(), 64, 64, 0, None) == 0  # nothing to do: no launch


@pytest.mark.parametrize("args", [
    (None, 64, 8, 2048, 128, 0, 1), (64, 8, 8, 2048, 128, 0, 1), (64, 64, 8, 2048, 120, 0, 1), (64, 64, 8, 2048, 132, 0, 1),
    (64, 64, 1 << 31, 2048, 128, 0, 1), (64, 64, 8, 2048, 128, 2, 1), (64, 64, 8, 2048, 128, 1, 2), (64, 64, 8, 2048, 128, 0, 0),
])
def test_write_refusals(args):
    k, v, held, layer_stride, row_stride, layer, layers = args
    assert _lib.load().xpu_kv_write(cache(), 64, 64, 1, 4, None, k, v, held, layer_stride, row_stride, layer, layers, None) == INVALID
    assert "xpu_kv_write" in _lib.last_error()


PROMPT = dict(dtype=0, plan=64, blocks=1, q=64, k=64, v=64, out=64, lse=None, tokens=8, q_heads=4, kv_heads=2, head_dim=64,
              q_stride=256, kv_stride=128, out_stride=256, scale=1.0)


@pytest.mark.parametrize("change,status", [
    ({"plan": None}, INVALID), ({"plan": 4}, INVALID), ({"q": None}, INVALID), ({"out": None}, INVALID), ({"k": 72}, INVALID),
    ({"dtype": 9}, INVALID), ({"kv_heads": 0}, INVALID), ({"q_heads": 5}, INVALID), ({"q_heads": 1}, INVALID),
    ({"head_dim": 80}, UNSUPPORTED), ({"q_heads": 130, "q_stride": 8320, "out_stride": 8320}, UNSUPPORTED),
    ({"q_stride": 252}, INVALID), ({"q_stride": 248}, INVALID), ({"kv_stride": 64}, INVALID), ({"out_stride": 128}, INVALID),
    ({"kv_stride": 1 << 38}, INVALID), ({"tokens": 1 << 31}, INVALID), ({"scale": 0.0}, INVALID), ({"scale": -1.0}, INVALID),
    ({"scale": float("inf")}, INVALID), ({"scale": float("nan")}, INVALID),
])
def test_prompt_refusals(change, status):
    assert _lib.load().xpu_prompt_attention(*(PROMPT | change).values(), None) == status
    assert "xpu_prompt_attention" in _lib.last_error()


def test_prompt_without_tokens_is_nothing_to_do():
    assert _lib.load().xpu_prompt_attention(*(PROMPT | {"tokens": 0}).values(), None) == 0


TREE = dict(layer=0, sequences=64, starts=64, ancestors=64, count=1, nodes=4, q=64, k=64, v=64, out=64, lse=None, q_heads=4,
            q_stride=256, kv_stride=128, out_stride=256, scale=1.0, workspace=64, workspace_bytes=1 << 40)


@pytest.mark.parametrize("change,status", [
    ({"layer": 2}, INVALID), ({"sequences": None}, INVALID), ({"starts": None}, INVALID), ({"ancestors": None}, INVALID),
    ({"count": 1025}, INVALID), ({"q": 72}, INVALID), ({"v": None}, INVALID), ({"q_heads": 3}, INVALID),
    ({"q_heads": 256, "q_stride": 1 << 14, "out_stride": 1 << 14}, UNSUPPORTED), ({"q_stride": 250}, INVALID),
    ({"workspace": None}, INVALID), ({"workspace": 8}, INVALID), ({"workspace_bytes": 0}, INVALID),
])
def test_tree_refusals(change, status):
    assert _lib.load().xpu_tree_attention(cache(), *(TREE | change).values(), None) == status
    assert "xpu_tree_attention" in _lib.last_error()


def plan(lens, q_heads, kv_heads, capacity=1 << 16):
    n = np.asarray(lens, np.uint32)
    out, used = np.full(capacity, -7, np.int32), ctypes.c_size_t()
    status = _lib.load().xpu_prompt_plan(n.ctypes.data, n.size, q_heads, kv_heads, out.ctypes.data, out.size, ctypes.byref(used))
    return status, out, used.value


@pytest.mark.parametrize("lens,q_heads,kv_heads", [([37], 32, 8), ([1, 0, 2047, 64, 65], 16, 8), ([8192], 32, 8), ([5] * 300, 7, 1),
                                                   ([0, 0], 4, 2), ([], 4, 4), ([200, 64], 64, 1), ([4096] * 2, 28, 4)])
def test_plan_covers_every_position_once(lens, q_heads, kv_heads):
    status, p, used = plan(lens, q_heads, kv_heads)
    assert status == 0
    blocks, tokens, items, group = p[:4]
    assert tokens == sum(lens) and group == q_heads // kv_heads and blocks <= max(items, 0)
    offsets = p[4:4 + blocks + 1]
    assert (np.diff(offsets) > 0).all() and offsets[0] == 0 and offsets[-1] == items
    at = (4 + blocks + 1 + 3) // 4 * 4
    assert used == at + 4 * items and (p[used:] == -7).all()
    span = 2 * (128 // group)
    seen = np.zeros((tokens, kv_heads), int)
    firsts = {int(a): n for a, n in zip(np.cumsum([0] + list(lens)), lens) if n}
    for token, length, pos, head in p[at:used].reshape(-1, 4):
        assert firsts[int(token)] == length and pos % span == 0 and pos < length
        seen[token + pos:token + min(pos + span, length), head] += 1
    assert (seen == 1).all()
    if items:  # no block has more than its share and the longest item
        cost = np.minimum(p[at:used].reshape(-1, 4)[:, 2] + span, p[at:used].reshape(-1, 4)[:, 1]) // 128 + 2
        load = [cost[offsets[b]:offsets[b + 1]].sum() for b in range(blocks)]
        assert max(load) <= cost.sum() / blocks + cost.max() + 1


def test_plan_refusals():
    status, _, used = plan([100], 4, 2, capacity=8)
    assert status == INVALID and used > 8
    L, n = _lib.load(), np.asarray([4], np.uint32)
    got = ctypes.c_size_t()
    assert L.xpu_prompt_plan(n.ctypes.data, 1, 3, 2, None, 0, ctypes.byref(got)) == INVALID
    assert L.xpu_prompt_plan(n.ctypes.data, 1, 130, 2, None, 0, ctypes.byref(got)) == UNSUPPORTED
    assert L.xpu_prompt_plan(None, 1, 2, 2, None, 0, ctypes.byref(got)) == INVALID
    big = np.asarray([0x7fffffff, 2], np.uint32)
    assert L.xpu_prompt_plan(big.ctypes.data, 2, 2, 2, None, 0, ctypes.byref(got)) == INVALID


def test_sizes():
    L = _lib.load()
    assert L.xpu_kv_workspace_size(10) >= 4 * 4 * 1024
    assert L.xpu_kv_workspace_size(100000) >= 4 * 4 * 100000
    assert L.xpu_tree_attention_workspace_size(1, 1, 4, 0, 64) == 0
    assert L.xpu_tree_attention_workspace_size(1, 1, 4, 2, 64) > 0
