"""Each form of the 8-bit products' kernel with whole and with shared tiles, for one matrix and by expert, in each output type. The form that a call
takes is looked up in the code that chooses it (tests/f8_walk.py), so a new choice cannot leave one of them out unseen."""
import pytest
import torch

import f8_exact as ex
import f8_walk
from test_gpu_f8 import TYPES, check, problem
from unpopped_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def expects(form, shared, m, n, k, begin):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert f8_walk.form(m, n, k, len(begin) - 1, sms) == form
    assert f8_walk.shared(form, begin, n, k, sms, f8_walk.panel_rows(k)) == shared


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k,form,shared", [
    (61, 4111, 2064, "narrow", False), (300, 300, 8192, "narrow", True),
    (384, 4096, 4096, "wide 128", False), (700, 2051, 2048, "wide 128", False), (513, 2051, 8192, "wide 128", True),
    (1100, 4096, 528, "wide 256", False), (2100, 4099, 512, "wide 256", False), (600, 4096, 8192, "wide 256", True),
    (2000, 2051, 8208, "pair 256", False), (4096, 2304, 4096, "pair 256", False), (5000, 512, 8192, "pair 256", True), (1100, 4111, 8208, "pair 256", True),
])
def test_one_matrix(m, n, k, form, shared, dtype):
    expects(form, shared, m, n, k, [0, m])
    x, xs, w, ws = problem(m + n, m, n, k)
    check(ops.f8_matmul(x, xs, w, ws, dtype=dtype), x, xs, w, ws)


def test_panels():
    m, n, k = 2100, 2049, 24576
    expects("pair 256", True, m, n, k, [0, m])
    assert m > f8_walk.panel_rows(k)
    x, xs, w, ws = problem(m, m, n, k)
    check(ops.f8_matmul(x, xs, w, ws, dtype=torch.float32), x, xs, w, ws)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes,n,k,form,shared", [
    ([3, 0, 40, 7], 1003, 2064, "narrow", False), ([5, 0, 60], 384, 16400, "narrow", True),
    ([200, 1300, 1500], 2048, 1024, "wide 128", False), ([600, 600], 2048, 8192, "wide 128", True),
    ([512, 512], 4096, 2048, "wide 256", False), ([1000, 1000], 4099, 4112, "wide 256", False),
    ([1500, 1400], 3001, 6160, "pair 256", False), ([1400, 1400], 4096, 8192, "pair 256", True), ([1300, 1300], 2050, 8208, "pair 256", True),
])
def test_by_expert(sizes, n, k, form, shared, dtype):
    begin = [0]
    for s in sizes:
        begin.append(begin[-1] + s)
    expects(form, shared, begin[-1], n, k, begin)
    x, xs, w, ws = problem(n + k, begin[-1], n, k, len(sizes))
    got = ops.f8_expert_matmul(x, xs, w, ws, torch.tensor(begin, dtype=torch.int32, device=DEV), dtype=dtype)
    for e, (lo, hi) in enumerate(zip(begin, begin[1:])):
        if hi > lo:
            check(got[lo:hi], x[lo:hi], xs[lo:hi], w[e], ws[e])


@pytest.mark.parametrize("sizes", [[100, 2000, 2000], [1792, 0, 1793, 1791]])
def test_panels_by_expert(sizes):
    """Some experts' rows are more than L2 is given, others' are not; every eighth row is looked at."""
    n, k = 4400, 24576
    begin = [0]
    for s in sizes:
        begin.append(begin[-1] + s)
    assert f8_walk.form(begin[-1], n, k, len(sizes)) != "narrow"
    assert max(sizes) > f8_walk.panel_rows(k) > min(s for s in sizes if s)
    x, xs, w, ws = problem(n, begin[-1], n, k, len(sizes))
    got = ops.f8_expert_matmul(x, xs, w, ws, torch.tensor(begin, dtype=torch.int32, device=DEV))
    for e, (lo, hi) in enumerate(zip(begin, begin[1:])):
        if hi > lo:
            check(got[lo:hi][::8], x[lo:hi][::8], xs[lo:hi][::8], w[e], ws[e])
    ops.check_workspace("f8", torch.device(DEV))
