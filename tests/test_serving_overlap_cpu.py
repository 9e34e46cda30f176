"""Gathered weights that lie in the cache's arrays are refused (no GPU)."""
import pytest

import kraken_hip as kh
from test_paged_cpu import cache_of, fake
from test_serving_cpu import gather, refused, vctx  # noqa: F401  (a fixture)

CODES, SCALES, MOVED = 5 * 64 * 2 * 256, 4 * 5 * 2, 4 * 3 * 2 * 90


@pytest.mark.parametrize("name,size", [("kp", CODES), ("vp", CODES), ("ks", SCALES),
                                       ("vs", SCALES)])
def test_gathered_weights_in_the_cache(vctx, name, size):  # noqa: F811
    cache = cache_of(**{name: fake(size, 0x700000)})
    for at in (0x700000, 0x700000 + size - 4, 0x700000 - MOVED + 4):
        refused(vctx, "gather_kv_pages_q8", gather(cache=cache, output=fake(MOVED, at)),
                "must not overlap")
    for at in (0x700000 + size, 0x700000 - MOVED):
        status = vctx.status("gather_kv_pages_q8", *gather(cache=cache, output=fake(MOVED, at)))
        assert status == kh.UNAVAILABLE, kh.last_error()
