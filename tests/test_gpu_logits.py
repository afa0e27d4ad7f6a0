"""The operators over rows of logits on the device, against the float64 oracle (tests/logits_cases.py
derives the tolerances)."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import numba_cuda_amd as cuda
from numba_cuda_amd import logits
from numba_cuda_amd.cudadrv import devicearray
from oracle import logits64
from tests import logits_cases as cases

KINDS = ["normal", "edge"]


# ---- adjust --------------------------------------------------------------------------------

@pytest.mark.parametrize("name", cases.DTYPES)
@pytest.mark.parametrize("rows, vocab, longest, pairs, mask", [
    (1, 1, 1, 0, None), (1, 5, 3, 1, "rows"), (3, 31, 200, 5, "shared"), (4, 4095, 1000, 0, "rows"),
    (5, 4096, 10, 300, "rows"), (2, 4097, 5000, 2, None), (7, 10007, 0, 0, "shared"), (4, 10007, 70000, 1500, "rows")])
def test_adjust(name, rows, vocab, longest, pairs, mask):
    cases.check_adjust(cuda, rows, vocab, name, name, longest, pairs, mask)
    cases.check_adjust(cuda, rows, vocab, name, "float32", longest, pairs, mask, index="int64", pad=5)
    cases.check_adjust(cuda, rows, vocab, name, name, longest, pairs, mask, per_row=False, in_place=True, pad=1)


@pytest.mark.parametrize("name", cases.DTYPES)
def test_adjust_of_special_rows(name):
    cases.check_adjust(cuda, 9, 5003, name, name, 800, 20, "rows", kind="edge")
    cases.check_adjust(cuda, 9, 5003, name, "float32", 800, 20, None, kind="edge")


def test_adjust_keeps_nan_apart_and_masks_it():
    x = np.float32([[np.nan, 1, np.inf, -np.inf] * 20])
    mask = np.uint32([[0xfffffff0, 0xffffffff, 0xffff]])
    got = logits.adjust(cuda.to_device(x), tokens=cuda.to_device(np.int32([0, 2, 6, 7, 5, 5])),
                        offsets=cuda.to_device(np.int32([0, 6])), repetition=2.0, presence=1.0, frequency=0.5,
                        mask=cuda.to_device(mask)).copy_to_host()[0]
    want = x[0].copy()
    want[:4] = -np.inf
    want[5] = 0.5 - 1.0 - 1.0
    assert np.array_equal(got, want, equal_nan=True)


def test_adjust_clamps_offsets_and_takes_host_arrays():
    x = np.ones((3, 10), np.float32)
    got = logits.adjust(x, tokens=[1, 2, 3], offsets=[-5, 2, 1, 99], presence=[1.0, 2.0, 3.0]).copy_to_host()
    want = np.ones((3, 10))
    want[0, [1, 2]] = 0              # tokens [0, 2)
    want[2, [2, 3]] = -2             # tokens [1, 3); row 1 is empty
    assert np.array_equal(got, want)


def test_adjust_leaves_what_lies_beside_the_rows():
    wide = np.arange(4 * 50, dtype=np.float32).reshape(4, 50)
    d = cuda.to_device(wide)
    logits.adjust(d[:, 7:40], d[:, 7:40], mask=cuda.to_device(np.zeros(2, np.uint32)))
    want = wide.copy()
    want[:, 7:40] = -np.inf
    assert np.array_equal(d.copy_to_host(), want)


# ---- top -----------------------------------------------------------------------------------

@pytest.mark.parametrize("name", cases.DTYPES)
@pytest.mark.parametrize("rows, vocab, k", [
    (1, 1, 1), (2, 7, 7), (3, 1000, 1), (3, 1000, 1000), (1, 4096, 50), (2, 8193, 64), (9, 20011, 257), (2, 40000, 1024),
    (1030, 300, 5), (600, 9001, 40)])
def test_top(name, rows, vocab, k):
    cases.check_top(cuda, rows, vocab, name, k, pad=3)
    cases.check_top(cuda, rows, vocab, name, k, lse=False, seed=1)


@pytest.mark.parametrize("name", cases.DTYPES)
@pytest.mark.parametrize("rows, vocab, k", [(8, 1001, 30), (8, 30011, 1), (8, 30011, 100), (8, 9000, 1024),
                                            (8, 100003, 1), (8, 100003, 100), (8, 100003, 700)])
def test_top_of_special_rows(name, rows, vocab, k):
    cases.check_top(cuda, rows, vocab, name, k, kind="edge")
    cases.check_top(cuda, rows, vocab, name, k, kind="edge", temperature=0.7)


@pytest.mark.parametrize("k", [3, 200])
def test_top_orders_nan_and_infinities(k):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((3, 20000)).astype(np.float32)
    x[0, ::97] = np.nan
    x[1, ::5] = np.inf
    x[1, 1::5] = -np.inf
    x[2, 5::2] = np.nan
    x.view(np.uint32)[2, 5::4] |= 0x80000000       # NaNs of both signs
    cases.check_top(cuda, 3, 20000, "float32", k, data=x)


def test_top_of_rows_that_fill_the_list_again_and_again():
    # upwards: every entry exceeds all before it; one workgroup per row, hundreds of cuts
    line = np.arange(150000, dtype=np.float32)
    x = np.concatenate([line[None], line[None, ::-1], np.repeat(line[::1000], 1000)[None, :150000]])
    x = np.repeat(x, 400, 0)
    d = cuda.to_device(x)
    for k in (1, 64, 1024):
        values, indices = logits.top(d, k)
        got = indices.copy_to_host()
        for r in range(3):
            want = logits64.top(x[r * 400:r * 400 + 1], k) if k == 64 else np.lexsort(
                (np.arange(150000), -x[r * 400]))[None, :k]
            assert np.array_equal(got[r * 400:(r + 1) * 400], np.repeat(want, 400, 0))


@pytest.mark.parametrize("vocab", [40000, 200000])
@pytest.mark.parametrize("k", [1, 50, 600])
def test_top_of_masked_rows(vocab, k):
    """Fewer entries than asked for are left: the rest are the first of the masked ones."""
    rng = np.random.default_rng(vocab + k)
    for left in (0, 1, 30, k):
        x = np.full((3, vocab), -np.inf, np.float32)
        for r in range(3):
            at = rng.permutation(vocab)[:left]
            x[r, at] = rng.standard_normal(left)
        cases.check_top(cuda, 3, vocab, "float32", k, data=x)


def test_top_into_wider_arrays_and_their_surroundings():
    rng = np.random.default_rng(9)
    x = rng.standard_normal((5, 6000)).astype(np.float16)
    values = cuda.to_device(np.full((5, 20), 7, np.float16))
    indices = cuda.to_device(np.full((5, 20), -7, np.int32))
    got = logits.top(cuda.to_device(x), 9, values=values[:, 3:12], indices=indices[:, 4:13])
    assert got[0].shape == (5, 9)
    want = logits64.top(x, 9)
    v, i = values.copy_to_host(), indices.copy_to_host()
    assert np.array_equal(i[:, 4:13], want) and (i[:, :4] == -7).all() and (i[:, 13:] == -7).all()
    assert np.array_equal(v[:, 3:12], np.take_along_axis(x, want, 1)) and (v[:, :3] == 7).all() and (v[:, 12:] == 7).all()


def test_rows_upside_down_and_repeated():
    rng = np.random.default_rng(10)
    x = rng.standard_normal((6, 5000)).astype(np.float32)
    d = cuda.to_device(x)
    upside = devicearray.DeviceNDArray((6, 5000), (-20000, 4), np.float32, gpu_data=d.gpu_data.view(5 * 20000))
    assert np.array_equal(logits.top(upside, 4)[1].copy_to_host(), logits64.top(x[::-1], 4))
    same = devicearray.DeviceNDArray((6, 5000), (0, 4), np.float32, gpu_data=d.gpu_data)
    assert np.array_equal(logits.top(same, 4)[1].copy_to_host(), np.repeat(logits64.top(x[:1], 4), 6, 0))


# ---- distillation --------------------------------------------------------------------------

@pytest.mark.parametrize("name", cases.DTYPES)
@pytest.mark.parametrize("what", ["loss", "both", "apart"])
@pytest.mark.parametrize("rows, vocab, k", [(1, 1, 1), (3, 5, 9), (5, 1009, 8), (2, 8193, 64), (7, 20011, 200),
                                            (3, 4096, 1024), (6, 30000, 0), (1100, 777, 5)])
def test_distill(name, what, rows, vocab, k):
    cases.check_distill(cuda, rows, vocab, name, k, what=what, pad=3)
    cases.check_distill(cuda, rows, vocab, name, k, what=what, temperature=2.0, full=k > 0, teacher=name, index="int64",
                        in_place=True)


@pytest.mark.parametrize("name", cases.DTYPES)
@pytest.mark.parametrize("what", ["both", "apart"])
def test_distill_of_special_rows_and_repeated_indices(name, what):
    cases.check_distill(cuda, 9, 9001, name, 50, what=what, kind="edge")
    cases.check_distill(cuda, 9, 301, name, 50, what=what, kind="edge", temperature=3.0)
    cases.check_distill(cuda, 6, 40, name, 300, what=what, repeated=True)
    cases.check_distill(cuda, 1200, 11, name, 30, what=what, repeated=True)


def test_rows_without_entries_and_with_nothing_allowed():
    x = np.float32([[1, 2, 3], [np.nan, 1, 2], [-np.inf] * 3, [-np.inf, 0, 0]])
    values = np.float32([[1, 2], [1, 2], [0, 0], [0, 0]])
    indices = np.int32([[-1, 3], [5, -2], [1, 1], [0, 1]])
    loss, lse, grad = (a.copy_to_host() for a in logits.distill_loss_and_grad(
        1.0, cuda.to_device(x), cuda.to_device(values), cuda.to_device(indices)))
    assert loss[0] == loss[1] == 0 and not grad[:2].any()            # no entry: nothing, even beside a NaN
    assert loss[2] == np.inf and np.array_equal(grad[2], [0, -1, 0])    # a row of -inf has q = 0
    assert loss[3] == np.inf and np.allclose(grad[3], [-0.5, 0, 0.5], atol=4 * cases.U)
    assert lse[2] == -np.inf and np.isnan(lse[1])


def test_gradient_of_a_broadcast_number():
    rng = np.random.default_rng(2)
    x, v = rng.standard_normal((4, 600)).astype(np.float32), rng.standard_normal((4, 3)).astype(np.float32)
    i = rng.integers(0, 600, (4, 3)).astype(np.int32)
    args = [cuda.to_device(a) for a in (x, v, i)]
    one = cuda.to_device(np.float32([0.25]))
    spread = devicearray.DeviceNDArray((4,), (0,), np.float32, gpu_data=one.gpu_data)
    for g in (0.25, spread, [0.25] * 4):
        got = logits.distill_loss_and_grad(g, *args)[2].copy_to_host()
        assert np.array_equal(got, logits.distill_loss_and_grad(cuda.to_device(np.full(4, 0.25, np.float32)),
                                                               *args)[2].copy_to_host())


def test_gradient_against_differences_of_the_loss():
    rng = np.random.default_rng(4)
    x = rng.standard_normal((2, 50)).astype(np.float32)
    v, i = rng.standard_normal((2, 4)).astype(np.float32), np.int32([[0, 7, 7, 49], [3, -1, 20, 11]])
    dv, di = cuda.to_device(v), cuda.to_device(i)
    weights = np.float32([1.0, -2.0])
    grad = logits.distill_loss_and_grad(cuda.to_device(weights), cuda.to_device(x), dv, di,
                                        temperature=1.5)[2].copy_to_host()
    step = np.float32(2.0 ** -6)
    moved = np.concatenate([x[r] + s * step * np.eye(50, dtype=np.float32) for s in (1, -1) for r in range(2)])
    loss, _ = logits.distill_loss(cuda.to_device(moved), cuda.to_device(np.tile(np.repeat(v, 50, 0), (2, 1))),
                                  cuda.to_device(np.tile(np.repeat(i, 50, 0), (2, 1))), temperature=1.5)
    loss = loss.copy_to_host().astype(np.float64).reshape(2, 2, 50)
    got = (loss[0] - loss[1]) / (2 * float(step)) * weights[:, None]
    # the loss is about 4 and off by some 40 roundings; third derivatives are below 1/10
    assert np.abs(got - grad).max() < 2 * (40 * cases.U * 4 / float(step) + float(step) ** 2 / 60)


# ---- as they are used ------------------------------------------------------------------------

def test_teacher_to_student():
    """adjust -> top -> distillation, on a stream, in bfloat16; then the student after a step."""
    rng = np.random.default_rng(6)
    rows, vocab, k = 40, 12007, 32
    teacher, tx = cases.rows_like(rng, rows, vocab, "bfloat16")
    student, sx = cases.rows_like(rng, rows, vocab, "bfloat16")
    mask = rng.integers(0, 2 ** 32, (rows, (vocab + 31) // 32), dtype=np.uint64).astype(np.uint32)
    tokens = rng.integers(0, vocab, 500).astype(np.int32)
    offsets = np.linspace(0, 500, rows + 1).astype(np.int64)
    s = cuda.stream()
    dt, ds = cuda.to_device(teacher, stream=s), cuda.to_device(student, stream=s)
    full = cuda.device_array((rows, vocab), np.float32, stream=s)
    logits.adjust(dt, full, tokens=cuda.to_device(tokens, stream=s), offsets=cuda.to_device(offsets, stream=s),
                  repetition=1.2, mask=cuda.to_device(mask, stream=s), stream=s)
    values, indices, norm = logits.top(full, k, lse=True, temperature=2.0, stream=s)
    loss, lse, grad = logits.distill_loss_and_grad(1.0 / rows, ds, values, indices, temperature=2.0, teacher_lse=norm,
                                                   stream=s)
    adjusted = full.copy_to_host(stream=s)
    s.synchronize()
    got_i, got_v, got_n = indices.copy_to_host(), values.copy_to_host(), norm.copy_to_host()
    s.synchronize()
    want_adjusted = logits64.adjust(tx, tokens, offsets, None, 1.2, allowed=cases.allowed_of(mask, vocab))
    cases.close(adjusted, want_adjusted, 3 * cases.U * np.where(np.isfinite(want_adjusted), np.abs(tx) * 1.2, 0), "adjust")
    assert np.array_equal(got_i, logits64.top(adjusted, k))
    want_loss, want_lse, want_grad = logits64.distill(sx, got_v, got_i, 2.0, got_n, np.full(rows, 1.0 / rows))
    cases.close(loss.copy_to_host(), want_loss, 1e-5 * (1 + np.abs(want_loss)), "loss")
    got_grad = cases.decode(grad.copy_to_host())
    s.synchronize()
    cases.close(got_grad, want_grad, 2.0 ** -8 * np.abs(want_grad) + 1e-6, "gradient")
    # against the gradient the loss falls
    moved, _ = cases.encode(sx - 20 * rows * got_grad, "float32")
    after, _ = logits.distill_loss(cuda.to_device(moved), values, indices, temperature=2.0, teacher_lse=norm)
    assert (after.copy_to_host() < want_loss).all()


def test_results_do_not_change_from_call_to_call():
    rng = np.random.default_rng(7)
    x = cuda.to_device(rng.standard_normal((70, 30001)).astype(np.float32))
    g = cuda.to_device(rng.random(70).astype(np.float32))
    first = None
    for _ in range(5):
        v, i, z = logits.top(x, 100, lse=True)
        now = [a.copy_to_host().tobytes() for a in (v, i, z, *logits.distill_loss_and_grad(g, x, v, i))]
        first = first or now
        assert now == first


def test_calls_on_several_streams_at_once():
    rng = np.random.default_rng(8)
    streams = [cuda.stream() for _ in range(4)]
    hosts = [rng.standard_normal((3, 60000)).astype(np.float32) for _ in streams]
    arrays = [cuda.to_device(h) for h in hosts]
    got = []
    for _ in range(10):
        for s, d in zip(streams, arrays):
            v, i = logits.top(d, 20, stream=s)
            got.append((s, v, i, logits.distill_loss(d, v, i, stream=s)[0]))
    cuda.synchronize()
    want = [logits64.top(h, 20) for h in hosts]
    losses = [logits64.distill(h, np.take_along_axis(h, w, 1), w)[0] for h, w in zip(hosts, want)]
    for n, (s, v, i, loss) in enumerate(got):
        assert np.array_equal(i.copy_to_host(), want[n % 4])
        s.synchronize()
        cases.close(loss.copy_to_host(), losses[n % 4], 1e-5, "loss")
        s.synchronize()


def test_torch_tensors_and_offsets_past_32_bits():
    torch = pytest.importorskip("torch")
    x = torch.randn(3, 5001, device="cuda").to(torch.bfloat16)
    values, indices = torch.empty(3, 4, dtype=torch.bfloat16, device="cuda"), torch.empty(3, 4, dtype=torch.int32,
                                                                                          device="cuda")
    got = logits.top(x[:, 1:], 4, values=values, indices=indices)
    assert got[0] is values
    assert np.array_equal(indices.cpu().numpy(), logits64.top(x[:, 1:].float().cpu().numpy(), 4))
    assert logits.top_workspace(1, 131072, 4, torch.bfloat16) == logits.top_workspace(1, 131072, 4, logits.bfloat16)
    # rows more than 4 GiB apart
    far = torch.zeros(5 << 30, dtype=torch.uint8, device="cuda")
    pitch = 2200000000
    rows = torch.as_strided(far.view(torch.float16), (3, 2001), (pitch // 2, 1))
    rows.copy_(torch.randn(3, 2001, device="cuda"))
    host = rows.cpu().numpy()
    assert np.array_equal(logits.top(rows, 10)[1].copy_to_host(), logits64.top(host, 10))
    logits.adjust(rows, rows, mask=cuda.to_device(np.full(63, 0xffff0000, np.uint32)))
    want = host.copy()
    want[:, np.arange(2001) % 32 < 16] = -np.inf
    assert np.array_equal(rows.cpu().numpy(), want)


def test_recorded_into_a_graph_and_replayed():
    torch = pytest.importorskip("torch")
    rows, vocab, k = 6, 60011, 20                # rows long enough that both calls need a workspace
    x = torch.zeros(rows, vocab, device="cuda")
    tokens = torch.randint(0, vocab, (300,), device="cuda", dtype=torch.int32)
    offsets = torch.arange(rows + 1, device="cuda") * 50
    y, grad = torch.empty_like(x), torch.empty_like(x)
    values, indices = torch.empty(rows, k, device="cuda"), torch.empty(rows, k, dtype=torch.int32, device="cuda")
    norm, loss, lse = (torch.empty(rows, device="cuda") for _ in range(3))
    space = torch.empty(max(logits.top_workspace(rows, vocab, k, np.float32),
                            logits.distill_workspace(rows, vocab, k, np.float32, grad=True)), dtype=torch.uint8,
                        device="cuda")

    def chain(stream, workspace):
        logits.adjust(x, y, tokens=tokens, offsets=offsets, repetition=1.1, frequency=0.1, stream=stream)
        logits.top(y, k, values=values, indices=indices, lse=norm, workspace=workspace, stream=stream)
        logits.distill_loss_and_grad(0.5, x, values, indices, teacher_lse=norm, loss=loss, lse=lse, out=grad,
                                     workspace=workspace, stream=stream)

    chain(0, space)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        stream = cuda.external_stream(torch.cuda.current_stream().cuda_stream)
        with pytest.raises(ValueError, match="captured"):
            logits.top(y, k, stream=stream)
        with pytest.raises(ValueError, match="needs a workspace"):
            logits.top(y, k, values=values, indices=indices, stream=stream)
        chain(stream, space)
    for n in range(4):
        x.copy_(torch.randn(rows, vocab, device="cuda") * (n + 1))
        graph.replay()
        torch.cuda.synchronize()
        recorded = [t.clone() for t in (y, values, indices, norm, loss, lse, grad)]
        for t in (y, values, indices, norm, loss, lse, grad):
            t.zero_()
        chain(0, None)                   # the same calls, eager, with the stream's own workspace
        torch.cuda.synchronize()
        for got, want in zip((y, values, indices, norm, loss, lse, grad), recorded):
            assert torch.equal(got, want)


@pytest.mark.parametrize("call", ["adjust", "top", "distill"])
def test_no_rows(call):
    x = cuda.device_array((0, 50), np.float32)
    if call == "adjust":
        assert logits.adjust(x).shape == (0, 50)
        assert logits.adjust(cuda.device_array((3, 0), np.float32)).shape == (3, 0)
    elif call == "top":
        assert [a.shape for a in logits.top(x, 3, lse=True)] == [(0, 3), (0, 3), (0,)]
    else:
        v, i = cuda.device_array((0, 3), np.float32), cuda.device_array((0, 3), np.int32)
        assert [a.shape for a in logits.distill_loss_and_grad(1.0, x, v, i)] == [(0,), (0,), (0, 50)]
        empty = logits.distill_loss_and_grad(1.0, cuda.device_array((2, 0), np.float32), cuda.to_device(
            np.zeros((2, 3), np.float32)), cuda.to_device(np.zeros((2, 3), np.int32)))
        assert not empty[0].copy_to_host().any() and (empty[1].copy_to_host() == -np.inf).all()


@pytest.mark.parametrize("name", cases.DTYPES)
@pytest.mark.parametrize("in_place, repeated", [(False, False), (True, True)])
def test_large_gradient_by_itself(name, in_place, repeated):
    rows, vocab = (1300, 27001) if name == "float32" else (2500, 27001)      # over 128 MiB: three launches
    assert logits.distill_workspace(rows, vocab, 20, cases.np_dtype(name), loss=False, grad=True) > 0
    cases.check_distill(cuda, rows, vocab, name, 20, what="apart", in_place=in_place, repeated=repeated,
                        pad=0 if in_place else 5, full=not repeated)


def test_large_gradient_of_special_rows():
    cases.check_distill(cuda, 1700, 20011, "float32", 6, what="apart", kind="edge", temperature=0.7)


def test_two_threads_on_one_stream():
    """Calls of several launches that share the stream's workspace, from two host threads."""
    import threading
    rng = np.random.default_rng(12)
    stream = cuda.stream()
    hosts = [rng.standard_normal((2, 100003)).astype(np.float32) for _ in range(2)]
    arrays = [cuda.to_device(h) for h in hosts]
    results, errors = [[], []], []

    def work(n):
        try:
            cuda.current_context()
            for _ in range(50):
                v, i, z = logits.top(arrays[n], 7, lse=True, stream=stream)
                results[n].append((i, z, logits.distill_loss(arrays[n], v, i, stream=stream)[0]))
        except Exception as error:      # noqa: BLE001
            errors.append(error)
    threads = [threading.Thread(target=work, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    stream.synchronize()
    for n, host in enumerate(hosts):
        want = logits64.top(host, 7)
        first = None
        for i, z, loss in results[n]:
            got = (i.copy_to_host(), z.copy_to_host(), loss.copy_to_host())
            stream.synchronize()
            assert np.array_equal(got[0], want)
            first = first or got
            assert np.array_equal(got[1], first[1]) and np.array_equal(got[2], first[2])


@pytest.mark.parametrize("name, vocab", [("float32", 524288), ("float32", 524289), ("bfloat16", 1048576), ("float16", 1500001)])
def test_very_long_rows(name, vocab):
    """At and past the number of entries from which a workgroup of top's first launch takes several pieces."""
    rng = np.random.default_rng(vocab)
    a, x = cases.rows_like(rng, 2, vocab, name)
    d = cuda.to_device(a)
    for k in (1, 1000):
        v, i, z = logits.top(d, k, lse=True)
        want = np.argsort(-x, axis=1, kind="stable")[:, :k]
        assert np.array_equal(i.copy_to_host(), want)
        assert np.abs(z.copy_to_host() - logits64.lse(x)).max() < 1e-5 * 30
    loss, lse, grad = logits.distill_loss_and_grad(1.0, d, v, i)
    wl, wz, wg = logits64.distill(x, cases.decode(v.copy_to_host()), want, 1.0, None, [1.0, 1.0])
    assert np.abs(loss.copy_to_host() - wl).max() < 1e-4 and np.abs(lse.copy_to_host() - wz).max() < 3e-4
    cases.close(cases.decode(grad.copy_to_host()), wg, cases.HALF_STEP[name] * np.abs(wg) + 1e-4 * np.abs(wg) + 1e-6, "gradient")


# rows about the lengths where a row is kept in registers and LDS in other shares, and read by more lanes
@pytest.mark.parametrize("name, around", [("float32", 4096), ("float32", 24576), ("float32", 32768),
                                          ("bfloat16", 16384), ("bfloat16", 49152), ("float16", 81920)])
def test_distill_of_rows_kept_in_part(name, around):
    for vocab in (around - 1, around, around + 1, around + 100):
        cases.check_distill(cuda, 3, vocab, name, 40, what="both", pad=5)
        cases.check_distill(cuda, 3, vocab, name, 1024, what="both", temperature=2.0, in_place=True)


@pytest.mark.parametrize("name, vocab", [("float32", 4099), ("float32", 16384), ("bfloat16", 8193), ("float16", 32768)])
def test_distill_of_many_rows(name, vocab):
    cases.check_distill(cuda, 520, vocab, name, 20, what="both", in_place=True)
    cases.check_distill(cuda, 520, vocab, name, 20, what="both", kind="edge", pad=1)


@pytest.mark.parametrize("name", cases.DTYPES)
@pytest.mark.parametrize("rows, vocab, k", [(2048, 1009, 64), (2500, 300, 1), (2048, 4096, 33), (2049, 3, 3), (1030, 600, 400),
                                            (1024, 9000, 300)])
def test_top_of_many_rows(name, rows, vocab, k):
    cases.check_top(cuda, rows, vocab, name, k, pad=5)
    cases.check_top(cuda, rows, vocab, name, k, kind="edge")


@pytest.mark.parametrize("k", [1, 10, 64])
def test_top_of_many_masked_rows(k):
    rng = np.random.default_rng(19)
    a = np.full((2100, 4000), np.finfo(np.float32).min, np.float32)
    a[1::3] = -np.inf
    a[2::3] = 1.5                                    # all alike
    for row in range(0, 2100, 7):
        a[row, rng.integers(0, 4000, row % 300)] = rng.standard_normal(row % 300)
    a[5] = np.arange(4000)
    a[6] = -np.arange(4000)
    values, indices = (o.copy_to_host() for o in logits.top(cuda.to_device(a), k)[:2])
    order = np.argsort(-a, axis=1, kind="stable")[:, :k]
    assert np.array_equal(indices, order)
    assert np.array_equal(values, np.take_along_axis(a, order, 1))


@pytest.mark.parametrize("name", cases.DTYPES)
@pytest.mark.parametrize("rows, vocab, longest, pairs", [(4, 900, 50, 5000), (3, 9000, 0, 9000), (2, 5000, 40000, 3000)])
def test_adjust_with_biases_for_all(name, rows, vocab, longest, pairs):
    cases.check_adjust(cuda, rows, vocab, name, name, longest, pairs, "rows")


@pytest.mark.parametrize("name", ["float32", "bfloat16"])
def test_distill_of_many_rows_and_entries(name):
    cases.check_distill(cuda, 300, 33000, name, 600, what="both", pad=3)
