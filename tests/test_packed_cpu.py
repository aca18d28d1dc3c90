"""What needs no GPU of a cache held in 4 bits: sizes, the pool, the settings, refusals, the plain format itself."""

import numpy as np
import pytest
import torch

from plain_packed import PackedCase, held, slab_bytes


@pytest.mark.parametrize("page,dim", [(16, 64), (1, 1), (1, 32), (2, 33), (4, 96), (64, 256), (8, 80)])
def test_slab_sizes(page, dim):
    from pagedserve_b200.cache.manager import CacheGroup, KVNeed
    from pagedserve_b200.kernels.ops import packed_slab_bytes

    slab = packed_slab_bytes(page, dim)
    assert slab == slab_bytes(page, dim) and slab % 16 == 0 and 0 <= slab - page * -(-dim // 32) * 20 < 16
    group = CacheGroup(KVNeed(3, dim), [4, 7], page, 5, 9, torch.float32, "cpu", scratch_pages=1, packed=True)
    assert group.pool.shape == (6, 2, 2, 3, slab) and group.pool.dtype == torch.uint8
    k, v = group.layer_views(7)
    assert k.shape == v.shape == (6, 3, slab) and k.stride() == (group.page_stride, slab, 1) == v.stride()
    assert group.bytes_per_page == group.page_stride == 2 * 2 * 3 * slab


def test_plain_groups():
    rng = np.random.default_rng(0)
    for size in (1, 5, 32, 40, 100):
        row = rng.normal(size=size).astype(np.float32)
        kept = held(row)
        for first in range(0, size, 32):
            x, y = row[first:first + 32], kept[first:first + 32]
            span = x.max() - x.min() + abs(x.min()) * 2.0 ** -7
            assert np.abs(x - y).max() <= 0.5 * span / 15 * (1 + 2.0 ** -7) + 1e-6
    assert (held(np.zeros(40)) == 0).all() and np.isnan(held(np.full(3, np.inf))).all()


def test_settings():
    from pagedserve_b200.config.engine_config import EngineConfig
    from pagedserve_b200.config.registry import ConfigError

    assert EngineConfig().kv_cache_dtype == "model" and EngineConfig(kv_cache_dtype="int4").kv_cache_dtype == "int4"
    with pytest.raises(ConfigError, match="int8"):
        EngineConfig(kv_cache_dtype="int8")


def test_layers_that_can_be_packed():
    """Which designs' caches can be held in 4 bits is said by their mixers."""
    from pagedserve_b200.config import gozunex, pagatar, suvunex, tefopel, vozirax, zositar
    from pagedserve_b200.config.gpt2 import named_config
    from pagedserve_b200.config.registry import resolve_architecture
    from pagedserve_b200.models.model import Model
    from pagedserve_b200.parts.base import PartEnv

    def packs(config):
        _, _, builder = resolve_architecture(config.to_dict())
        model = Model(builder(config), PartEnv(ops=None, dtype=torch.float32, device="cpu"))
        return all(block.mixer.packs_cache for block in model.blocks if block.mixer.cache_need() is not None)

    assert packs(named_config("tiny-a"))
    assert packs(zositar.named_config("zositar-tiny")) and packs(tefopel.named_config("tefopel-tiny"))
    assert not packs(gozunex.named_config("gozunex-tiny")) and not packs(vozirax.named_config("vozirax-tiny"))
    assert not packs(pagatar.named_config("pagatar-tiny")) and not packs(suvunex.named_config("suvunex-tiny"))


def test_tensors_on_the_host_are_refused():
    """The wrappers look at every argument before anything is launched."""
    from pagedserve_b200.kernels.ops import KernelError, Ops

    ops = Ops(torch.float32)
    case = PackedCase([20], 2, 64, 16, torch.float32)
    planes = (case.pool[:, 0], case.pool[:, 1], case.pool.stride(0))
    rows = case.k.flatten(1)
    with pytest.raises(KernelError, match="CUDA device"):
        ops.kv_append_packed(rows, rows, case.token_row, case.positions, case.table, *planes, 2, 64, 16)
    with pytest.raises(KernelError, match="CUDA device"):
        ops.packed_attention_tokens(rows, rows, *planes, case.token_row, case.positions, case.table, 2, 2, 64, 16, None, 0.1, 20)
    with pytest.raises(KernelError, match="pages of a power of two"):
        ops.packed_attention_tokens(rows, rows, *planes, case.token_row, case.positions, case.table, 2, 2, 300, 16, None, 0.1, 20)
    with pytest.raises(KernelError, match="CUDA device"):
        ops.token_logprobs(torch.zeros(2, 10), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(KernelError, match="CUDA device"):
        ops.head_logprobs(torch.zeros(2, 8), torch.zeros(10, 8), torch.zeros(2, dtype=torch.int32))


def test_counts_beyond_32_bits_are_refused():
    """(kernels count rows and columns in 32 bits: a larger number would be cut without a word)"""
    from pagedserve_b200.kernels.ops import KernelError, Ops

    ops, targets = Ops(torch.float32), torch.zeros(1, dtype=torch.int32)
    for rows, vocabulary in ((2 ** 31 - 1, 10), (1, 2 ** 31 - 1), (1, 2 ** 32 + 5)):
        with pytest.raises(KernelError, match="of up to"):
            ops._logprob_results("token_logprobs", rows, vocabulary, targets, 0, targets.get_device())


def test_declared_arguments_are_the_sources():
    """(a call whose declaration is one argument short passes a number where a stream is meant)"""
    import ctypes
    import re
    from pathlib import Path

    from pagedserve_b200.kernels import build, ops

    declared = ops._SIGNATURES["packed"]
    kinds = {ctypes.c_void_p: "P", ctypes.c_int: "I", ctypes.c_longlong: "L", ctypes.c_float: "F"}
    found = {}
    for name in build.LIBRARIES["packed"]:
        text = (Path(build.__file__).parent.parent / "csrc" / name).read_text()
        for entry in re.finditer(r"PS_EXPORT int (\w+)\(([^)]*)\)", text):
            found[entry[1]] = "".join("P" if "*" in part else "L" if "long long" in part else "F" if "float" in part else "I" for part in entry[2].split(","))
    assert found == {name: "".join(kinds[kind] for kind in arguments) for name, arguments in declared.items()}


def test_shares_of_prompts():
    """Clusters only while every CTA has an SM of its own, and no share of fewer than two tiles."""
    from pagedserve_b200.kernels.ops import Ops

    for n_items, queries, longest, extent, heads in ((1, 64, 64, 0, 12), (1, 128, 4000, 0, 12), (2, 2048, 1024, 0, 12), (1, 1024, 1024, 0, 25), (3, 2048, 8192, 0, 16),
                                                     (1, 64, 1, 0, 1), (5, 64, 70, 20, 3), (1, 64, 10 ** 6, 0, 8), (1, 64, 10 ** 6, 100, 8), (200, 12800, 64, 0, 64)):
        blocks = (queries // 64 + 3 * n_items) // 4
        shares, most = Ops._prompt_shares(n_items, blocks, queries, longest, extent, heads)
        assert shares in (1, 2, 4, 8) and most >= 1
        assert shares == 1 or (most >= 2 and heads * blocks <= 148)
    assert Ops._prompt_shares(1, 1, 128, 4000, 0, 12) == (8, 4) and Ops._prompt_shares(1, 4, 1024, 1024, 0, 25)[0] == 1
