"""Two host threads that call one entry point with different sizes at a time: a
kernel's limit of shared memory, which a launch of one thread needs, is not lowered
by the other's call."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from tinygnn_b200 import _lib
    return _lib.lib


def rand(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def together(calls, rounds):
    """Runs each of the calls (of a stream) `rounds` times in a thread of its own, all at a time; the statuses other than 0."""
    start, bad, streams = threading.Barrier(len(calls)), [], [torch.cuda.Stream() for _ in calls]

    def work(k):
        start.wait()
        for i in range(rounds):
            status = calls[k](streams[k].cuda_stream)
            if status:
                bad.append((k, i, status))
                return
            if i % 100 == 99:
                streams[k].synchronize()
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return bad


def distill(lib, rows, classes, k):
    from tinygnn_b200 import _lib
    z, teacher = rand(rows, classes, seed=k), rand(rows, k, seed=k + 1)
    ids = torch.arange(rows * k, device="cuda", dtype=torch.int32).view(rows, k) % classes
    loss, dz = torch.empty(rows, device="cuda"), torch.empty_like(z)

    def call(stream):
        return lib.tg_distill_loss(rows, classes, _lib.F32, z.data_ptr(), classes, k, ids.data_ptr(), 4, k, _lib.F32, teacher.data_ptr(), k,
                                   2.0, None, loss.data_ptr(), dz.data_ptr(), classes, stream)
    return call, (loss, dz), (z, teacher, ids)


@pytest.mark.parametrize("classes,ks", [(16, (128, 64)), (41, (128, 96)), (1000, (8, 128)), (20000, (8, 8))])
def test_distillation_of_different_sizes(lib, classes, ks):
    """Narrow rows with few and many entries; rows of a warp, and of a cluster, of two widths."""
    sides = [distill(lib, 200 if classes < 5000 else 20, classes if n == 0 else classes + (0 if classes < 300 else classes // 2), k)
             for n, k in enumerate(ks)]
    want = []
    for call, out, _ in sides:
        assert call(torch.cuda.current_stream().cuda_stream) == 0
        want.append([t.clone() for t in out])
    assert together([s[0] for s in sides], 1500) == []
    for (_, out, _), ref in zip(sides, want):
        assert all(torch.equal(a, b) for a, b in zip(out, ref))


def test_group_norm_of_different_sizes(lib):
    from tinygnn_b200 import _lib
    rows, cols, graphs = 64, 2048, 8
    x = rand(rows, cols, seed=1, dtype=torch.bfloat16)
    gamma, beta = rand(cols, seed=2), rand(cols, seed=3)
    off = torch.arange(0, rows + 1, rows // graphs, device="cuda", dtype=torch.int32)
    calls, results = [], []
    for groups in (1, 256):
        y, dx, dg, db = torch.empty_like(x), torch.empty_like(x), torch.empty_like(gamma), torch.empty_like(gamma)
        stats = torch.empty(graphs, groups, 2, device="cuda")

        def call(stream, groups=groups, y=y, dx=dx, dg=dg, db=db, stats=stats):
            status = lib.tg_group_norm(rows, cols, groups, graphs, off.data_ptr(), _lib.BF16, x.data_ptr(), cols, _lib.F32, gamma.data_ptr(),
                                       beta.data_ptr(), 1e-5, 0, 0.0, y.data_ptr(), cols, stats.data_ptr(), stream)
            return status or lib.tg_group_norm_grad(rows, cols, groups, graphs, off.data_ptr(), _lib.BF16, x.data_ptr(), cols, x.data_ptr(),
                                                    cols, stats.data_ptr(), _lib.F32, gamma.data_ptr(), beta.data_ptr(), 0, 0.0,
                                                    dx.data_ptr(), cols, dg.data_ptr(), db.data_ptr(), stream)
        calls.append(call)
        results.append((y, stats, dx, dg, db))
    want = []
    for call, out in zip(calls, results):
        assert call(torch.cuda.current_stream().cuda_stream) == 0
        want.append([t.clone() for t in out])
    assert together(calls, 1500) == []
    for out, ref in zip(results, want):
        assert all(torch.equal(a, b) for a, b in zip(out, ref))


def test_degree_order_of_different_sizes(lib):
    calls, results = [], []
    for rows in (300000, 1000):
        ptr = torch.cat([torch.zeros(1), torch.rand(rows, generator=torch.Generator().manual_seed(rows)).mul(9).floor().cumsum(0)]).int().cuda()
        out = torch.empty(rows, dtype=torch.int32, device="cuda")
        calls.append(lambda stream, rows=rows, ptr=ptr, out=out: lib.tg_csr_degree_order(rows, ptr.data_ptr(), out.data_ptr(), stream))
        results.append(out)
    want = []
    for call, out in zip(calls, results):
        assert call(torch.cuda.current_stream().cuda_stream) == 0
        want.append(out.clone())
    assert together(calls, 1500) == []
    assert all(torch.equal(out, ref) for out, ref in zip(results, want))
