"""The order of the numbers inside one page of one kv head.

The cache tensors keep their logical shapes (keys ``[..., P, d]``, values
``[..., d, P]``), but the ``P * d`` numbers of a (page, kv head) pair lie in the
order in which the attention kernels' matrix-core fragments read them, so that
every wave instruction reads consecutive memory:

* keys:   ``[16-key block][octet of d][key in block][8]``
* values: ``[16-key block][16-wide block of d][group of 4 keys][number in block][4]``

(the same formulas as ``kcache_index`` / ``vcache_index`` in ``csrc/common.h``).
The kernels never need this module; it serves tests, tools and anyone who wants
to look into a cache from Python.

The windowed attention with a sink keeps its keys row by row (``[..., P, D]``) and its
values ``[..., P, E]`` in the order ``[P / 4][E][4]`` (the four keys of a quad side by side
for each value channel): ``value_quads`` gives that view.

A cache of 8-bit keys and values (e4m3 codes, ``kv_scale [..., 2, P]`` one byte for every key and value) has the logical
shapes of the first one and an order of its own, in which 16 consecutive bytes are one lane's share of a load:

* keys:   ``[16-key block][sixteen of d][key in block][16]``
* values: ``[16-key block][group of four 16-wide blocks of d][group of 4 keys][number in block][block of the group][4]``
  (the last group may hold fewer than four blocks)

(``key_index`` / ``value_index`` in ``csrc/e4m3_cache.hip``): ``e4m3_key_index``, ``e4m3_value_index``, and
``e4m3_numbers``, what a cache holds as float32 numbers.
"""
from __future__ import annotations

import torch


def key_index(page_size: int, d: int) -> torch.Tensor:
    """``[P, d]`` int64: where key ``k``'s number ``dd`` lies in the flat page."""
    k = torch.arange(page_size).view(-1, 1)
    dd = torch.arange(d).view(1, -1)
    return (((k >> 4) * (d >> 3) + (dd >> 3)) * 16 + (k & 15)) * 8 + (dd & 7)


def value_index(page_size: int, d: int) -> torch.Tensor:
    """``[d, P]`` int64: where number ``dd`` of the value of key ``k`` lies."""
    k = torch.arange(page_size).view(1, -1)
    dd = torch.arange(d).view(-1, 1)
    return ((((k >> 4) * (d >> 4) + (dd >> 4)) * 4 + ((k & 15) >> 2)) * 16 + (dd & 15)) * 4 + (k & 3)


def _scatter(logical: torch.Tensor, index: torch.Tensor) -> torch.Tensor:
    flat = logical.reshape(*logical.shape[:-2], -1)
    out = torch.empty_like(flat)
    out[..., index.reshape(-1).to(flat.device)] = flat
    return out.view(logical.shape)


def _gather(physical: torch.Tensor, index: torch.Tensor) -> torch.Tensor:
    flat = physical.reshape(*physical.shape[:-2], -1)
    return flat[..., index.reshape(-1).to(flat.device)].view(physical.shape)


def keys_to_cache_order(keys: torch.Tensor) -> torch.Tensor:
    """``[..., P, d]`` row-major keys -> the same shape in cache order."""
    return _scatter(keys, key_index(keys.shape[-2], keys.shape[-1]))


def keys_from_cache_order(keys: torch.Tensor) -> torch.Tensor:
    return _gather(keys, key_index(keys.shape[-2], keys.shape[-1]))


def values_to_cache_order(values: torch.Tensor) -> torch.Tensor:
    """``[..., d, P]`` transposed values -> the same shape in cache order."""
    return _scatter(values, value_index(values.shape[-1], values.shape[-2]))


def values_from_cache_order(values: torch.Tensor) -> torch.Tensor:
    return _gather(values, value_index(values.shape[-1], values.shape[-2]))


def value_quads(values: torch.Tensor) -> torch.Tensor:
    """``[..., P, E]`` pages of the windowed attention's values as ``[..., P / 4, E, 4]``: entry
    ``[..., o >> 2, e, o & 3]`` is channel ``e`` of the value of the key at offset ``o``."""
    p, e = values.shape[-2], values.shape[-1]
    return values.view(*values.shape[:-2], p // 4, e, 4)


def e4m3_key_index(page_size: int, d: int) -> torch.Tensor:
    """``[P, d]`` int64: where the code of key ``k``'s number ``dd`` lies in the flat page."""
    k = torch.arange(page_size).view(-1, 1)
    dd = torch.arange(d).view(1, -1)
    return (((k >> 4) * (d >> 4) + (dd >> 4)) * 16 + (k & 15)) * 16 + (dd & 15)


def e4m3_value_index(page_size: int, d: int) -> torch.Tensor:
    """``[d, P]`` int64: where the code of number ``dd`` of the value of key ``k`` lies."""
    k = torch.arange(page_size).view(1, -1)
    dd = torch.arange(d).view(-1, 1)
    wide = torch.clamp((d >> 4) - 4 * (dd >> 6), max=4)
    return ((k >> 4) * 16 * d + (dd >> 6) * 1024
            + ((((k & 15) >> 2) * 16 + (dd & 15)) * wide + ((dd >> 4) & 3)) * 4 + (k & 3))


def e4m3_numbers(k_cache: torch.Tensor, v_cache: torch.Tensor, kv_scale: torch.Tensor):
    """The float32 keys ``[..., P, d]`` and values ``[..., d, P]`` that pages of 8 bits stand for."""
    page_size, d = k_cache.shape[-2], k_cache.shape[-1]
    size = (kv_scale.to(torch.int32) << 23).view(torch.float32)
    k = _gather(k_cache.view(torch.uint8), e4m3_key_index(page_size, d)).view(torch.float8_e4m3fn).float()
    v = _gather(v_cache.view(torch.uint8), e4m3_value_index(page_size, d)).view(torch.float8_e4m3fn).float()
    return k * size[..., 0, :].unsqueeze(-1), v * size[..., 1, :].unsqueeze(-2)
