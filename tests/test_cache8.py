"""The 8-bit cache on the host: which models may have one, what it takes, what is refused without a device; the plain rounding against torch's."""

import pytest
import torch

from gtar_kimik3_public_b200.cache import Cache, CacheLayout
from gtar_kimik3_public_b200.generate import parse_cache_dtype
from gtar_kimik3_public_b200.models.model import Model
from gtar_kimik3_public_b200.ops.functional import KernelError, PagedKV8, rows8_cut, rows8_wins
from gtar_kimik3_public_b200.parts.base import KVRequest, StateRequest
from gtar_kimik3_public_b200.registry import architecture, config_from_dict
from tests.dasusun_configs import DAS_CONFIGS
from tests.katopel_configs import KAT_CONFIGS
from tests.plain import cache8 as plain8
from tests.pofadra_configs import POF_CONFIGS
from tests.rezulorn_configs import REZ_CONFIGS
from tests.tiny_configs import TINY_A
from tests.topezen_configs import TPZ_CONFIGS
from tests.zasorax_configs import ZAS_CONFIGS

E4 = torch.float8_e4m3fn


def model_of(raw, **options):
    config = config_from_dict(raw)
    return Model(architecture(config.ARCH_NAMES[0]).build_plan(config), config, torch.bfloat16, "cpu", **options)


def test_names_of_the_cache_dtype():
    assert parse_cache_dtype(None) is None and parse_cache_dtype("auto") is None
    assert parse_cache_dtype("float8_e4m3fn") is E4 and parse_cache_dtype(E4) is E4
    for wrong in ("float8", "int8", torch.float8_e5m2, torch.bfloat16):
        with pytest.raises(ValueError, match="cache_dtype"):
            parse_cache_dtype(wrong)


def test_requests_of_a_model_with_an_8_bit_cache():
    model = model_of(TINY_A, cache_dtype=E4)
    assert all(r.dtype is E4 for r in model.cache_layout().requests)
    assert all(r.dtype is None for r in model_of(TINY_A).cache_layout().requests)
    cache = model.make_cache(256)
    group, = cache.kv_groups
    assert group.k.dtype is E4 and group.v.dtype is E4 and group.k_exp.dtype is torch.uint8
    assert group.k_exp.shape == group.k.shape[:-1]
    layers, n_kv, d = TINY_A["num_hidden_layers"], TINY_A["num_key_value_heads"], TINY_A["head_dim"]
    assert cache.kv_bytes_per_token() == layers * n_kv * 2 * (d + 1)
    assert cache.scratch_bytes_per_token() == 4 * n_kv * d and model_of(TINY_A).make_cache(256).scratch_bytes_per_token() == 0


@pytest.mark.parametrize("raw", [DAS_CONFIGS["das_a"], POF_CONFIGS["pof_a"], POF_CONFIGS["pof_delta"], REZ_CONFIGS["rez_a"], ZAS_CONFIGS["zas_a"],
                                 TPZ_CONFIGS["tpz_a"], KAT_CONFIGS["kat_a"], KAT_CONFIGS["kat_delta"]])
def test_models_that_cannot(raw):
    model_of(raw)
    with pytest.raises(ValueError, match="grouped-query attention"):
        model_of(raw, cache_dtype=E4)


def test_refused_without_a_device():
    with pytest.raises(KernelError, match="B200"):
        PagedKV8(torch.zeros((1, 1, 64, 64), dtype=E4), torch.zeros((1, 1, 64, 64), dtype=E4), torch.zeros((1, 1, 64), dtype=torch.uint8),
                 torch.zeros((1, 1, 64), dtype=torch.uint8), torch.zeros((1, 1), dtype=torch.int32))
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        model_of(TINY_A, cache_dtype=torch.float16)


def test_requests_that_a_cache_refuses():
    for request in (KVRequest(2, 16, dtype=torch.float8_e5m2), KVRequest(2, 16, value_dim=32, dtype=E4)):
        with pytest.raises(ValueError, match="float8_e4m3fn"):
            Cache(CacheLayout([request]), 256, torch.bfloat16, "cpu")


def test_groups_of_both_kinds_beside_each_other():
    cache = Cache(CacheLayout([KVRequest(2, 16, dtype=E4), KVRequest(2, 16), [KVRequest(2, 16, window=100, dtype=E4), StateRequest((3,))]]), 64 * 6,
                  torch.bfloat16, "cpu", max_seqs=2)
    assert len(cache.kv_groups) == 3 and [g.request.dtype for g in cache.kv_groups] == [E4, None, E4]
    slot = cache.open()
    cache.grow(slot, 300)
    cache.check_invariants()
    cache.close(slot)
    cache.check_invariants()


def test_plain_rounding_is_the_type_s():
    y = torch.cat([torch.randn(4000, generator=torch.Generator().manual_seed(1), dtype=torch.float64) * 2.0 ** k for k in range(-8, 7)]).clamp(-448, 448)
    y = torch.cat([y, torch.arange(-4096, 4096, dtype=torch.float64) * 2.0**-13, torch.arange(-7168, 7169, dtype=torch.float64) / 16]).float().double()
    assert torch.equal(plain8.nearest8(y), y.float().to(E4).double())


def test_plain_powers():
    rows = torch.tensor([[0.0], [448.0], [448.5], [224.0], [224.25], [2.0**-80], [3.3895313892515355e38], [float("inf")]], dtype=torch.float64)
    assert plain8.exponent_of(rows).tolist() == [-64, 0, 1, -1, 0, -64, 119, -64]


PLACES = (444, 222, 111, 50)


def test_cuts_are_what_the_kernel_takes():
    for places in (PLACES, (296, 148, 71, 33)):
        for pairs in (1, 2, 7, 8, 64, 200, 512, 4096):
            for length in (0, 1, 31, 33, 200, 2000, 40000, 1 << 20):
                splits, pieces = rows8_cut(pairs, length, places)
                assert (splits in (1, 2, 4, 8) and pieces == 0) or (splits == 0 and places[0] // 2 <= pieces < places[0])
                assert splits <= max(1, -(-length // 32))


def test_cuts_at_measured_points():
    """Sequences x 8 kv heads: what was fastest, or within a few hundredths of it."""
    want = {(1, 4000): (8, 0), (4, 4000): (8, 0), (8, 500): (4, 0), (8, 1000): (4, 0), (16, 1000): (2, 0), (16, 2000): (2, 0), (24, 4000): (2, 0),
            (32, 1000): (1, 0), (48, 4000): (1, 0), (64, 4000): (2, 0), (96, 1000): (1, 0)}
    assert {k: rows8_cut(k[0] * 8, k[1], PLACES) for k in want} == want
    assert rows8_cut(8, 131072, PLACES)[0] == 0  # one long document: pieces


def test_prompts_through_few_rows_or_through_clean_pages():
    few = lambda n, new, past, n_kv=8, group=4, d=128: rows8_wins(n * new, n, new, past + new, n_kv, group, d, 148)  # noqa: E731
    assert few(16, 4, 2000) and few(16, 16, 2000) and few(1, 64, 4000) and few(1, 128, 0) and few(8, 32, 4000, 4, 3, 64)
    assert not few(16, 32, 2000) and not few(1, 512, 2000) and not few(1, 2048, 0) and not few(1, 2048, 0, 4, 3, 64)
    assert not few(4096, 64, 0)  # more row tiles than a grid has
