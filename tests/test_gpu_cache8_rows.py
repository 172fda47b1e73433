"""Rows on their way into the 8-bit cache that are not ordinary ones, in every kernel that writes."""

import pytest
import torch

from tests.plain import model as plain
from tests.test_gpu_cache8 import DEV, F, empty_pages, held, ints, rand

pytestmark = pytest.mark.gpu


def tables(positions, d):
    cos, sin = plain.rotary_tables(torch.arange(positions), d, 1e4)
    return cos[:, : d // 2].float().contiguous(), sin[:, : d // 2].float().contiguous()


@pytest.mark.parametrize("n_q,n_kv,d", [(4, 2, 128), (6, 2, 64)])
def test_a_position_outside_the_rotation_s_table(n_q, n_kv, d):
    """The decode kernel leaves such a token's key where it was, writes its value and reports it, as the write by itself does; the others are what they are."""
    lens = [65, 40, 90]
    cos, sin = (t.to(DEV) for t in tables(64, d))
    qkv = rand(3, (n_q + 2 * n_kv) * d, seed=7).to(torch.bfloat16).to(DEV)
    w = (1 + 0.1 * rand(d, seed=20)).float().to(DEV)
    pages = []
    for fused in (True, False):
        kv, slots, table = empty_pages(3, max(lens), n_kv, d)
        if fused:
            F().attention_decode8_fused(qkv, n_q, n_kv, d, w, w, 1e-6, cos, sin, kv, ints(*lens), slots, 63, max(lens), 0.1)
        else:
            F().qk_norm_rope_write8(qkv, n_q, n_kv, d, w, w, 1e-6, cos, sin, ints(*[m - 1 for m in lens]), ints(0, 1, 2), slots, kv, 63)
        with pytest.raises(Exception, match="page number"):
            F().check_kernel_errors(DEV)
        pages.append(kv)
        k, _ = held(kv, table, int(slots[0]), 65)
        assert torch.isnan(k[64]).all()  # the poison
    for name in ("k", "v", "k_exp", "v_exp"):
        assert torch.equal(getattr(pages[0], name).view(torch.uint8), getattr(pages[1], name).view(torch.uint8)), name
