"""Limits of the plans over the fp16 page pool: refused where their counts pass what the launches hold, the largest of 31 bits
among them.  Over the device without a GPU."""
import pytest

from rstr import hip
from test_pool_ops_refusals import dev, fake_lib, pool, pytestmark  # noqa: F401


@pytest.mark.parametrize("pages", [2 ** 31 - 1, 2 ** 31 - 16, 2 ** 31 - 31])
def test_selections_over_the_widest_tables(dev, pages):  # noqa: F811
    with hip.Session(0) as s:
        b = hip.BlockBounds(pool(s, n_kv=1))
        with pytest.raises(hip.RstrError, match="too many rows or pages") as e:
            hip.BlockSelect(b, 4, 1, 1, pages)
        assert e.value.code == -1
        hip.BlockSelect(b, 4, 1, 1, 2 ** 31 - 64).close()


@pytest.mark.parametrize("n_q,most", [(24, 2 ** 23 - 1), (16, 2 ** 24 - 17), (32, 2 ** 23 - 1)])
def test_plans_of_the_most_rows(dev, n_q, most):  # noqa: F811
    """One kv head: items of 16 columns of all tokens (and one a sequence), and of lists one for every 16 query heads that begin."""
    with hip.Session(0) as s:
        p = pool(s, n_kv=1)
        hip.PagedAttention(p, n_q, 1, most).close()
        for rows in (most + 17, 2 ** 24):
            with pytest.raises(hip.RstrError, match="too many rows") as e:
                hip.PagedAttention(p, n_q, 1, rows)
            assert e.value.code == -1
