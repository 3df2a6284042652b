"""The work that tracing reports of attention: products over the pairs that its band shows."""
import pytest

from sequences import visible
from test_gpu_attention import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('queries,keys', [(50, 60), (60, 50), (1, 40), (7, 1), (33, 33), (5, 0), (0, 5)])
@pytest.mark.parametrize('left,right', [(-1, -1), (-1, 0), (0, -1), (3, 2), (0, 0), (100, 0), (2, 100), (-1, 1 << 30)])
def test_work_is_the_visible_pairs(device, queries, keys, left, right):
    c = Case('bf16', 2, queries, keys, 4, 2, 64)
    device.trace(True)
    c.run(device, left, right)
    report = device.trace_report()
    device.trace(False)
    pairs = 2 * 4 * int(visible(queries, keys, queries, keys, left, right).sum())
    for name, products in (('attention', 2), ('attention_gradient', 5)):
        if name in report:  # (no queries: no forward)
            assert report[name][2] == 2 * products * 64 * pairs
    assert 'attention' in report or queries == 0
