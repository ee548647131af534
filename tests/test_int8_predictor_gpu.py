"""Runtime predictors with 8-bit hidden layers, and the retraining step of the hidden layers, through the analyzer's API."""
import numpy as np
import pytest
import torch

from habitat_b200 import batched, dense, workloads
from habitat_b200.analysis.mlp.mlp import RuntimePredictor, state_to_arrays
from oracle import mlp as omlp

pytestmark = pytest.mark.gpu


def _quantized(x):
    amax = np.abs(x).max(axis=1)
    with np.errstate(all="ignore"):
        q = np.rint(x * np.where(amax > 0, np.float32(127) / amax, np.float32(0))[:, None])
    return q, (amax / np.float32(127)).astype(np.float32)


def _replay(w, feats, dev, table, mu, sigma):
    """The 8-bit network in numpy with the kernels' roundings: multiply-adds of fc1 rounded once each, exact integer sums,
    float32 behind them; the last sum in float64.  -> predictions and the size of the last sum's terms."""
    x = np.concatenate([feats.astype(np.float64), table[dev]], axis=1)
    x = ((x - mu) / sigma).astype(np.float32)
    y = np.broadcast_to(w["fc1_b"], (len(x), len(w["fc1_b"]))).astype(np.float32)
    for c in range(x.shape[1]):
        # a product of two float32 numbers is exact in float64
        y = (y.astype(np.float64) + w["fc1_w"][:, c].astype(np.float64) * x[:, c:c + 1].astype(np.float64)).astype(np.float32)
    q, s = _quantized(np.maximum(y, 0))
    for hw, hb in zip(w["hidden_w"], w["hidden_b"]):
        qw, sw = _quantized(hw)
        y = (q.astype(np.float64) @ qw.astype(np.float64).T).astype(np.float32) * sw * s[:, None] + hb
        q, s = _quantized(np.maximum(y, 0))
    terms = q.astype(np.float64) * w["fc2_w"].astype(np.float64)
    return terms.sum(axis=1) * s + float(w["fc2_b"][0]), np.abs(terms).sum(axis=1) * s


def _weights(op, width=1024, layers=8, seed=0, gain=True):
    torch.manual_seed(seed)
    pred = RuntimePredictor(op, layers, width)
    w = state_to_arrays(pred.model)
    if gain:
        w["hidden_w"] = w["hidden_w"] * np.float32(6 ** 0.5)      # keeps the spread of the activations
    return {k: np.ascontiguousarray(v) for k, v in w.items()}


@pytest.mark.parametrize("op, width, layers, Q", [("linear", 1024, 8, 1), ("conv2d", 1024, 8, 16), ("lstm", 1024, 8, 17), ("bmm", 1024, 8, 700),
                                                  ("conv2d", 500, 3, 300), ("linear", 37, 1, 5), ("bmm", 1024, 2, 5000)])
def test_against_its_own_arithmetic(op, width, layers, Q):
    w = _weights(op, width, layers, Q)
    feats, dev = workloads.make_queries(op, Q, seed=Q)
    mu, sigma = workloads.batch_mu_sigma(*workloads.make_queries(op, 2000, seed=1))
    h = batched.Int8MLPHandle(feats.shape[1], mu=mu, sigma=sigma, device_features=workloads.BENCH_DEVICE_FEATURES, **w)
    got = h.predict(torch.from_numpy(feats).cuda(), torch.from_numpy(dev).cuda()).cpu().numpy()
    h.check_status()
    want, size = _replay(w, feats, dev, np.asarray(workloads.BENCH_DEVICE_FEATURES), mu, sigma)
    # the last sum: 1,024 terms through a tree of depth 32 + 5, each addition off by half a unit of at most the terms' sum
    assert (np.abs(got - want) <= 40 * 2.0 ** -24 * (size + np.abs(want))).all()


def test_in_pieces_and_with_a_result_given():
    w = _weights("linear", 256, 2)
    feats, dev = workloads.make_queries("linear", 1000, seed=3)
    mu, sigma = workloads.batch_mu_sigma(feats, dev)
    h = batched.Int8MLPHandle(feats.shape[1], mu=mu, sigma=sigma, device_features=workloads.BENCH_DEVICE_FEATURES, **w)
    f, d = torch.from_numpy(feats).cuda(), torch.from_numpy(dev).cuda()
    want = h.predict(f, d)
    h.chunk = 300
    out = torch.full((1000,), -1.0, device="cuda")
    assert h.predict(f, d, out) is out and torch.equal(out, want)
    assert np.array_equal(h.predict_host(feats, dev), want.cpu().numpy())
    assert h.predict_one(feats[7].tolist(), int(dev[7])) == float(want[7])
    assert h.predict(f[:0], d[:0]).shape == (0,)
    for bad in (lambda: h.predict(f[:, :3].contiguous(), d), lambda: h.predict(f, d[:5]), lambda: h.predict(f, d, out[:10]),
                lambda: h.predict_one([1.0], 0)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        h.predict(f.double(), d)


def test_close_to_the_float32_network():
    """Rounding to 8 bits is off by amax / 127 / sqrt(12) (rms).  Rows behind a ReLU: half of a normal distribution, rms sigma /
    sqrt(2), and the largest of 1,024 at about 3.3 sigma = 4.6 rms: 4.6 / 440 = 1.05 % of the row's rms.  Weights: uniform up to
    amax, rms amax / sqrt(3): 0.39 %.  A layer passes its input's error on as it does the input (the gain keeps the
    spread), so nine roundings of rows and eight of weights add up to sqrt(9 x 1.05^2 + 8 x 0.39^2) = 3.3 % of the last rows'
    size, which fc2 weighs like the rows themselves: sqrt(sum (w h)^2).  Half as much again is allowed.  (Not of the
    predictions' spread: most of a row is the same for all queries.)"""
    w = _weights("conv2d", seed=5)
    feats, dev = workloads.make_queries("conv2d", 2000, seed=6)
    mu, sigma = workloads.batch_mu_sigma(feats, dev)
    table = np.asarray(workloads.BENCH_DEVICE_FEATURES)
    h = batched.Int8MLPHandle(feats.shape[1], mu=mu, sigma=sigma, device_features=table, **w)
    got = h.predict_host(feats, dev).astype(np.float64)
    y = (np.concatenate([feats.astype(np.float64), table[dev]], axis=1) - mu) / sigma
    y = np.maximum(y @ w["fc1_w"].T.astype(np.float64) + w["fc1_b"], 0)
    for hw, hb in zip(w["hidden_w"], w["hidden_b"]):
        y = np.maximum(y @ hw.T.astype(np.float64) + hb, 0)
    terms = y * w["fc2_w"]
    want = terms.sum(axis=1) + float(w["fc2_b"][0])
    assert np.allclose(want, omlp.predict(w, feats, dev, table, mu, sigma), rtol=0, atol=1e-4 * np.abs(terms).sum(axis=1).max())
    assert np.sqrt(((got - want) ** 2).mean()) <= 1.5 * 0.033 * np.sqrt((terms ** 2).sum(axis=1).mean())


def test_predictor_precision_and_trace(monkeypatch):
    from habitat_b200.analysis import Device
    from habitat_b200.analysis.arguments import Arguments
    from habitat_b200.analysis.operation import MeasuredOperation
    from habitat_b200.analysis.predictor import Predictor
    from habitat_b200.analysis.run_time import RunTimeMeasurement
    from habitat_b200.analysis.trace import Trace
    monkeypatch.setenv("HABITAT_B200_PRECISION", "int8")
    predictor = Predictor()
    assert predictor._precision == "int8"
    torch.manual_seed(3)
    pred = RuntimePredictor("linear", 2, 128, precision="int8")
    pred.model.fc2.bias.data.fill_(50.0)                  # predicted times are positive
    pred.mu, pred.sigma = np.zeros(8), np.full(8, 1e4)
    predictor.linear_pred = pred
    plain = RuntimePredictor("linear", 2, 128, precision="bf16x3")
    plain.model.load_state_dict(pred.model.state_dict())
    plain.mu, plain.sigma = pred.mu, pred.sigma
    value, close = pred.predict([1, 64, 512, 256], "V100"), plain.predict([1, 64, 512, 256], "V100")
    assert isinstance(value, float) and abs(value - close) <= 0.02 * abs(close)
    # a trace: the operation's measured time by the ratio of the predictions (predictor.py:132-148 of the reference)
    operation = MeasuredOperation("linear", Arguments(((64, 512), (256, 512), None), {}), RunTimeMeasurement(3.0, [], Device.V100), None, Device.V100)
    there = {d: 3.0 * pred.predict([0, 64, 512, 256], d.name) / pred.predict([0, 64, 512, 256], "V100") for d in (Device.T4, Device.P100)}
    traces = Trace(Device.V100, [operation]).to_devices(list(there), predictor)
    for device, trace in zip(there, traces):
        assert abs(trace.run_time_ms - there[device]) <= 1e-6 * there[device]


def test_retrained_and_served_in_8_bits():
    """A run as it is used: a batch's gradients, a step of the hidden layers, predictions of the new weights in 8 bits."""
    torch.manual_seed(7)
    width, layers = 256, 3
    pred = RuntimePredictor("linear", layers, width, precision="int8")
    pred.model.cuda()
    feats, dev = workloads.make_queries("linear", 512, seed=8)
    pred.mu, pred.sigma = (np.concatenate([m[:4], [1e4] * 4]) for m in workloads.batch_mu_sigma(feats, dev))
    x = torch.randn(512, 8, device="cuda")
    before = [b.weight.detach().clone() for b in pred.model.mlp.layers if hasattr(b, "weight")]
    momentum = [torch.zeros_like(w) for w in before]
    for step, kwargs in enumerate((dict(), dict(nesterov=False, weight_decay=0.1))):
        pred.model.zero_grad()
        (pred.model(x) - x.sum(dim=1, keepdim=True)).square().mean().backward()
        grads = [b.weight.grad.clone() for b in pred.model.mlp.layers if hasattr(b, "weight")]
        rest = {n: p.detach().clone() for n, p in pred.model.named_parameters() if not n.startswith("mlp.") or n.endswith("bias")}
        pred.update_hidden(lr=0.02, **kwargs)
        for n, p in pred.model.named_parameters():
            if n in rest:
                assert torch.equal(p, rest[n])
        after = [b.weight.detach() for b in pred.model.mlp.layers if hasattr(b, "weight")]
        for i, (w, m, g) in enumerate(zip(before, momentum, grads)):
            m.mul_(0.95).add_(g)
            u = (g.double() + 0.95 * m.double()) if step == 0 else m.double()
            u = u / (u.norm() + 1e-7)
            for _ in range(5):
                a = u @ u.T
                u = 3.4445 * u + (-4.7750 * a + 2.0315 * (a @ a)) @ u
            want = (1.0 if step == 0 else 1.0 - 0.02 * 0.1) * w.double() - 0.02 * u
            # the update to float32's accuracy (1e-5 of it), the weights' own rounding
            assert float((after[i].double() - want).norm()) <= 0.02 * 1e-5 * float(u.norm()) + 2.0 ** -23 * float(want.norm())
        before = [w.detach().clone() for w in after]
    w = state_to_arrays(pred.model)
    got = pred.predict_batch(torch.from_numpy(feats).cuda(), torch.zeros(512, dtype=torch.uint8, device="cuda")).cpu().numpy()
    names = sorted(pred._device_rows)
    from habitat_b200.analysis.mlp.devices import get_all_devices
    table = np.array([get_all_devices(pred.device_params)[n] for n in names])
    want, size = _replay(w, feats, np.zeros(512, np.uint8), table, np.asarray(pred.mu, np.float64), np.asarray(pred.sigma, np.float64))
    assert (np.abs(got - want) <= 40 * 2.0 ** -24 * (size + np.abs(want))).all()


def test_update_refuses():
    pred = RuntimePredictor("linear", 2, 64)
    with pytest.raises(RuntimeError, match="gradients"):
        pred.update_hidden(0.1)
    pred.model(torch.randn(4, 8)).sum().backward()
    with pytest.raises(RuntimeError, match="GPU"):
        pred.update_hidden(0.1)
