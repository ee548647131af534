"""What an 8-bit predictor owes its caller beyond the numbers: its memory, its errors, its weights' updates."""
import ctypes

import numpy as np
import pytest
import torch

from habitat_b200 import _native, batched, dense, workloads
from habitat_b200.analysis.mlp.mlp import RuntimePredictor, state_to_arrays

pytestmark = pytest.mark.gpu


def _handle(width=256, layers=3, Q=600, op="linear", seed=1):
    torch.manual_seed(seed)
    w = state_to_arrays(RuntimePredictor(op, layers, width).model)
    feats, dev = workloads.make_queries(op, Q, seed=seed)
    mu, sigma = workloads.batch_mu_sigma(feats, dev)
    h = batched.Int8MLPHandle(feats.shape[1], mu=mu, sigma=sigma, device_features=workloads.BENCH_DEVICE_FEATURES, **w)
    return h, torch.from_numpy(feats).cuda(), torch.from_numpy(dev).cuda()


def _overwrite():
    """Takes what the allocator has free on the current stream in blocks of every size up to 4 MB, and fills it."""
    held = []
    for size in (512, 1024, 2048, 4096, 16384, 65536, 262144, 1048576, 4194304):
        held += [torch.full((size,), 85, dtype=torch.uint8, device="cuda") for _ in range(40)]
    return held


@pytest.mark.parametrize("captured", [False, True])
def test_weights_stay_until_queued_predictions_have_ended(captured):
    """A prediction waits on a stream of its own while the handle is dropped and its memory asked for again."""
    h, f, d = _handle()
    want = h.predict(f, d)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = h.predict(f, d)
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)          # some 0.1 s
        if captured:
            graph.replay()
        else:
            got = h.predict(f, d)
    del h
    held = _overwrite()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    del held


def test_closed():
    h, f, d = _handle()
    want = h.predict(f, d)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
        got = h.predict(f, d)
    h.close()
    held = _overwrite()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    del held
    h.close()
    for call in (lambda: h.predict(f, d), lambda: h.predict_host(f.cpu().numpy(), d.cpu().numpy()), lambda: h.predict_one([1.0] * 4, 0)):
        with pytest.raises(_native.HabitatNativeError, match="closed"):
            call()
    h.check_status()


def test_retrained_under_queued_predictions():
    """The same through the predictor: an update drops the pack and the next prediction uploads another."""
    torch.manual_seed(2)
    pred = RuntimePredictor("linear", 2, 128, precision="int8")
    pred.model.cuda()
    pred.mu, pred.sigma = np.zeros(8), np.full(8, 1e4)
    feats, dev = (torch.from_numpy(a).cuda() for a in workloads.make_queries("linear", 300, seed=4))
    want = pred.predict_batch(feats, dev).clone()
    pred.model(torch.randn(64, 8, device="cuda")).square().mean().backward()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
        got = pred.predict_batch(feats, dev)
    pred.update_hidden(0.5)
    new = pred.predict_batch(feats, dev)
    held = _overwrite()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and not torch.equal(new, want)
    del held


def _trained(seed=3, precision="int8", steps=1):
    """A predictor with gradients, after some updates."""
    torch.manual_seed(seed)
    pred = RuntimePredictor("linear", 2, 128, precision=precision)
    pred.model.cuda()
    pred.mu, pred.sigma = np.zeros(8), np.full(8, 1e4)
    x = torch.randn(64, 8, device="cuda")
    for _ in range(steps):
        pred.model.zero_grad()
        pred.model(x).square().mean().backward()
        pred.update_hidden(0.1)
    pred.model.zero_grad()
    pred.model(x).square().mean().backward()
    return pred


def _weights(pred):
    return [p.detach().clone() for p in pred.model.parameters()]


@pytest.mark.parametrize("failure", ["status", "steps"])
@pytest.mark.parametrize("nesterov", [True, False])
def test_an_update_that_raises_leaves_everything_as_it_was(failure, nesterov):
    pred, other = _trained(), _trained()
    before = _weights(pred)
    if failure == "status":
        _native.check(_native.load().hb_dense_inject_status(0x511))
    with pytest.raises(_native.HabitatNativeError):
        pred.update_hidden(0.1, nesterov=nesterov, steps=5 if failure == "status" else 0)
    assert all(torch.equal(a, b) for a, b in zip(before, _weights(pred)))
    for p in (pred, other):
        p.update_hidden(0.1, nesterov=nesterov)
    assert all(torch.equal(a, b) for a, b in zip(_weights(pred), _weights(other)))


# -- launches that gave up: the word as a kernel leaves it, written from the host ----------------

def _gives_up(code=0x531):
    torch.cuda.synchronize()
    _native.check(_native.load().hb_dense_inject_status(code))


def _other_call():
    dense.quantize_rows(torch.ones((2, 16), device="cuda"))
    dense.orthogonalize(torch.ones((4, 4), device="cuda"))


def test_a_failure_that_another_call_reported_is_not_lost_to_the_handle():
    h, f, d = _handle()
    h.predict(f, d)
    _gives_up()
    with pytest.raises(_native.HabitatNativeError, match="gave up"):
        _other_call()
    _other_call()                                     # told once
    with pytest.raises(_native.HabitatNativeError, match="gave up"):
        h.check_status()
    h.check_status()
    h.predict(f, d)
    h.check_status()


def test_every_handle_learns_of_a_failure_and_none_twice():
    h, f, d = _handle()
    other, _, _ = _handle(seed=2)
    h.predict(f, d), other.predict(f, d)
    _gives_up()
    for each in (h, other):
        with pytest.raises(_native.HabitatNativeError, match="gave up"):
            each.check_status()
    h.predict(f, d), other.predict(f, d)
    h.check_status(), other.check_status()
    late, _, _ = _handle(seed=3)
    late.predict(f, d)
    late.check_status()                               # of before its time
    _gives_up()
    with pytest.raises(_native.HabitatNativeError, match="gave up"):
        h.predict(f, d)
    h.predict(f, d)
    h.check_status()                                  # its predict has said so
    assert np.isfinite(h.predict_host(f.cpu().numpy(), d.cpu().numpy())).all()
    for each in (other, late):
        with pytest.raises(_native.HabitatNativeError, match="gave up"):
            each.check_status()


def test_every_thread_learns_of_a_failure():
    import threading
    dense.check_status()
    heard = []

    def look():
        try:
            dense.check_status()
            heard.append(False)
        except _native.HabitatNativeError:
            heard.append(True)
    count = dense.failures()
    _gives_up()
    for _ in range(2):                                # the first to look is told, a thread that starts afterwards is not
        t = threading.Thread(target=look)
        t.start()
        t.join()
    assert heard == [True, False] and dense.failures() == count + 1
    with pytest.raises(_native.HabitatNativeError, match="gave up"):
        dense.check_status()
    dense.check_status()
    dense.check_since(count + 1)
    with pytest.raises(_native.HabitatNativeError, match="gave up"):
        dense.check_since(count)


@pytest.mark.parametrize("precision", ["bf16", "bf16x3", "int8"])
@pytest.mark.parametrize("told", [False, True])
@pytest.mark.parametrize("how", ["predict", "save"])
def test_updates_that_gave_up_are_neither_served_nor_saved(precision, told, how, tmp_path):
    pred = _trained(precision=precision, steps=2)
    _gives_up()
    if told:
        with pytest.raises(_native.HabitatNativeError):
            _other_call()
    feats, dev = (torch.from_numpy(a).cuda() for a in workloads.make_queries("linear", 20, seed=4))
    path = str(tmp_path / "model.pth")
    for _ in range(2):
        with pytest.raises(_native.HabitatNativeError, match="gave up"):
            pred.predict_batch(feats, dev) if how == "predict" else pred.save_state(path)
    assert not (tmp_path / "model.pth").exists()
    with pytest.raises(_native.HabitatNativeError, match="gave up"):
        pred.update_hidden(0.1)
    pred.invalidate()                                 # the caller says that the weights are good
    pred.save_state(path)
    pred.load_state(path)
    assert bool(torch.isfinite(pred.predict_batch(feats, dev)).all())
    dense.check_status()


def test_features_are_divided_by_sigma():
    """The quotient rounded to float32, as in the other predictors, not a product with 1 / sigma: features whose quotient lies half-way between two
    float32 numbers, where the two differ."""
    rng = np.random.default_rng(1)
    cases = []
    while len(cases) < 40:
        x = np.float32(rng.uniform(1.0, 1000.0))
        half_way = (2 * int(rng.integers(2 ** 23, 2 ** 24)) + 1) * 2.0 ** -24       # 25 bits
        sigma = float(x) / half_way
        if np.float32(float(x) / sigma) != np.float32(float(x) * (1.0 / sigma)):
            cases.append((x, sigma))
    lib, p = _native.load(), lambda t: ctypes.c_void_p(t.data_ptr())
    f64 = lambda a: torch.tensor(a, dtype=torch.float64, device="cuda")
    w, b, devices, mu = torch.zeros((1, 5), device="cuda"), torch.zeros((1,), device="cuda"), f64([[1.0] * 4]), f64([0.0] * 5)
    w[0, 0] = 1.0
    row, q = torch.zeros((1,), dtype=torch.uint8, device="cuda"), torch.empty((1, 16), dtype=torch.int8, device="cuda")
    for x, sigma in cases:
        scales, feature, sigmas = torch.empty((1,), device="cuda"), torch.tensor([x], device="cuda"), f64([sigma] + [1.0] * 4)
        _native.check(lib.hb_int8_mlp_input(p(feature), 1, p(row), p(devices), 1, p(mu), p(sigmas), p(w), p(b), 1, 1, p(q), 16, p(scales),
                                            _native.current_stream_ptr()))
        # one feature through a weight of one: the row's scale is the quotient / 127
        assert float(scales) == np.float32(float(x) / sigma) / np.float32(127), (x, sigma)


def test_invalidate_does_not_hide_an_update_that_gave_up():
    """It belongs behind every change of weights, a step of the caller's optimizer after update_hidden for one."""
    pred = _trained(precision="bf16", steps=2)
    _gives_up()
    pred.invalidate()
    with pytest.raises(_native.HabitatNativeError, match="gave up"):
        pred.device_row("V100")


@pytest.mark.parametrize("precision", ["bf16", "int8"])
def test_traces_are_not_predicted_with_an_update_that_gave_up(precision):
    """Predictions of traces start their predictors early and try again where that raises."""
    from habitat_b200.analysis import Device
    from habitat_b200.analysis.arguments import Arguments
    from habitat_b200.analysis.operation import MeasuredOperation
    from habitat_b200.analysis.predictor import Predictor
    from habitat_b200.analysis.run_time import RunTimeMeasurement
    from habitat_b200.analysis.trace import Trace
    predictor = Predictor(precision=precision)
    predictor.linear_pred = _trained(precision=precision, steps=2)
    _gives_up()
    operation = MeasuredOperation("linear", Arguments(((64, 512), (256, 512), None), {}), RunTimeMeasurement(3.0, [], Device.V100), None, Device.V100)
    for _ in range(2):
        with pytest.raises(_native.HabitatNativeError, match="gave up"):
            Trace(Device.V100, [operation]).to_devices([Device.T4, Device.P100], predictor)
    predictor.linear_pred.invalidate()
    Trace(Device.V100, [operation]).to_devices([Device.T4, Device.P100], predictor)


def test_a_failure_that_another_threads_prediction_reported_is_not_lost():
    import threading
    h, f, d = _handle()
    h.predict(f, d)
    _gives_up()
    raised = []

    def other():
        dense.quantize_rows(torch.ones((2, 16), device="cuda"))
        for _ in range(2):
            try:
                h.predict(f, d)
                raised.append(False)
            except _native.HabitatNativeError:
                raised.append(True)
    t = threading.Thread(target=other)
    t.start()
    t.join()
    assert raised == [True, False]
    with pytest.raises(_native.HabitatNativeError, match="gave up"):
        h.check_status()
    h.check_status()


def test_results_carry_no_gradient():
    x = torch.randn(40, 64, device="cuda", requires_grad=True)
    q, scales = dense.quantize_rows(x)
    for y in (scales, dense.int8_matmul(q, scales, q, scales, bias=scales.detach().requires_grad_()), dense.orthogonalize(x)):
        assert not y.requires_grad and y.grad_fn is None
    assert "carry no gradient" in dense.__doc__
