"""The commit of kept rows counts every entry without a page once, also of a row that stays where it is."""
import numpy as np
import pytest

from rivoli_amd import hip
from tests.gpu_util import back, dev, dzeros

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("keys", [False, True])
@pytest.mark.parametrize("layers", [1, 3])
def test_rows_that_stay_are_counted_when_they_have_no_page(keys, layers):
    rng = np.random.default_rng(layers)
    page, n_pages, width = 16, 6, 64
    row_bytes = 2 * width if keys else width
    bytes_ = page * (row_bytes + (0 if keys else 4))
    pool = rng.integers(0, 256, (layers, n_pages, bytes_), dtype=np.uint8)
    # rows 14, 15 | 16 .. 31 | 32 ..: the first without pages; the second between two with them; the third past its table; the fourth whole
    tables = np.array([[-1, -1, n_pages], [0, -1, 1], [2, 2 ** 30, -7], [3, 4, 5]], np.int32)
    ctx = np.array([14, 14, 46, 14], np.int32)
    path = np.tile(np.arange(20, dtype=np.int32), (4, 1))
    n_path = np.array([4, 20, 3, 20], np.int32)
    path[1, 18:] = 19, 0                                  # rows 33 -> 32, both on a page; and one from before its place
    bad = 4 + (16 + 1) + 3
    want = pool.copy()
    for l in range(layers):
        p = want[l, 1]
        p[0:row_bytes] = pool[l, 1, row_bytes:2 * row_bytes]
        if not keys:
            p[page * row_bytes:][:4] = pool[l, 1, page * row_bytes + 4:][:4]
    launch = hip.launch_index_commit_paged if keys else hip.launch_kv_commit_paged
    for counted in (dzeros(4), None):
        pool_d, lens = dev(pool), dzeros(16, 0xEE)
        launch(pool_d, dev(tables), dev(ctx), dev(path), dev(n_path), 4, 20, 3, width, page, n_pages, layers, n_pages * page if keys else n_pages * bytes_, lens, counted)
        assert np.array_equal(back(pool_d), want.reshape(-1))
        assert np.array_equal(back(lens, np.int32), ctx + n_path)
        assert counted is None or int(back(counted, np.uint32)[0]) == bad
