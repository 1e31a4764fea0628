"""The edges of the 8-bit cache's operators: values and scales far apart, pages that are not there, lists that contradict themselves, many calls in a row."""
import numpy as np
import pytest

import cache_reference as ref
from deepforge_b200 import cache
from deepforge_b200.dfgpu import I32, tensor
from test_gpu_cache import ints, pages_state

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


# ---- pages

@pytest.mark.parametrize("op", ["reserve", "compact"])
def test_page_operations_one_behind_the_other(op):
    """Nothing but chained launches on the stream: each CTA of a launch finds the others of its cluster running before it writes to them."""
    rng = np.random.default_rng(3)
    state = pages_state(rng, 64, 9, 3000, 16, [], empty=(0,))
    grow = rng.integers(0, 40, (64, 1))
    want = ref.Pages(state.table, state.lengths, state.refs, [], 16)
    report = want.reserve([int(x) for x in grow[:, 0]]) if op == "reserve" else want.compact()
    p = cache.CachePagesParams(op=cache.PAGE_OPS[op], block=16)
    p.page_table, p.lengths, p.refs = tensor(I32, [64, 1, 9, 1]), tensor(I32, [64, 1, 1, 1]), tensor(I32, [3000])
    if op == "reserve":
        p.list = tensor(I32, [64, 1])
    ins = [ints(x) for x in (state.table, state.lengths, state.refs)]
    entries, calls = ints(grow), 300
    outs = [torch.full((calls, *x.shape), -99, device="cuda", dtype=torch.int32) for x in (*ins, ints([0] * 4))]
    scratch = torch.full((cache.query("cache_pages", p).scratch_bytes,), 255, device="cuda", dtype=torch.uint8)
    for i in range(calls):
        cache.cache_pages(p, [x.data_ptr() for x in ins] + [entries.data_ptr() if op == "reserve" else None] + [x[i].data_ptr() for x in outs], scratch.data_ptr())
    torch.cuda.synchronize()
    for got, expected in zip(outs, (want.table, want.lengths, want.refs, report)):
        assert bool((got == ints(expected)).all())
