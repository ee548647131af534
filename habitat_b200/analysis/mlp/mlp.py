"""MLP runtime predictors: the reference's load / save / predict API on the B200 kernel.

Reference: analyzer/habitat/analysis/mlp/mlp.py.  The torch modules keep the
reference's attribute names (fc1, mlp.layers.{0,2,...}, fc2, features) so its
checkpoints ({"mu", "sigma", "model": state_dict}, mlp.py:133-146) load
unchanged.  The modules only hold parameters: inference runs in the fused
sm_100a kernel (habitat_b200/csrc/mlp_chain.cu) through `predict_batch`, and
`predict` is that path with one query.  The reference's training loop
(mlp.py:148-250) is not here; `update_hidden` is the step of the hidden layers for a loop of
the caller's.
"""
import functools

import numpy as np
import torch
import torch.nn as nn

from habitat_b200.analysis.mlp.devices import get_all_devices, get_device_features

FEATURES = {
    "linear": ["bias", "batch", "in_features", "out_features"],
    "lstm": ["bias", "bidirectional", "batch", "seq_len", "input_size", "hidden_size",
             "num_layers"],
    "conv2d": ["bias", "batch", "image_size", "in_channels", "out_channels", "kernel_size",
               "stride", "padding"],
    "bmm": ["batch", "left", "middle", "right"],
}


class MLPBase(nn.Module):
    """`layers` x [Linear(layer_size, layer_size), ReLU] (mlp.py:17-31)."""

    def __init__(self, layers, layer_size):
        super().__init__()
        blocks = []
        for _ in range(layers):
            blocks += [nn.Linear(layer_size, layer_size), nn.ReLU()]
        self.layers = nn.ModuleList(blocks)

    def forward(self, x):
        for block in self.layers:
            x = block(x)
        return x


class _OpMLP(nn.Module):
    """fc1 (F + 4 -> layer_size) + ReLU, MLPBase, fc2 (layer_size -> 1); mlp.py:34-109."""

    op_name = None

    def __init__(self, layers, layer_size):
        super().__init__()
        self.features = list(FEATURES[self.op_name])
        self.fc1 = nn.Linear(len(self.features) + 4, layer_size)
        self.mlp = MLPBase(layers, layer_size)
        self.fc2 = nn.Linear(layer_size, 1)

    def forward(self, x):
        return self.fc2(self.mlp(torch.relu(self.fc1(x))))


class LinearMLP(_OpMLP):
    op_name = "linear"


class LSTMMLP(_OpMLP):
    op_name = "lstm"


class Conv2DMLP(_OpMLP):
    op_name = "conv2d"


class BMMMLP(_OpMLP):
    op_name = "bmm"


_MODEL_CLASSES = {"linear": LinearMLP, "lstm": LSTMMLP, "conv2d": Conv2DMLP, "bmm": BMMMLP}


def state_to_arrays(model):
    """Weights of an _OpMLP as the numpy arrays the native library packs."""
    sd = {k: v.detach().cpu().float().numpy() for k, v in model.state_dict().items()}
    n_hidden = len(model.mlp.layers) // 2
    return dict(
        fc1_w=sd["fc1.weight"], fc1_b=sd["fc1.bias"],
        hidden_w=np.stack([sd["mlp.layers.%d.weight" % (2 * i)] for i in range(n_hidden)]),
        hidden_b=np.stack([sd["mlp.layers.%d.bias" % (2 * i)] for i in range(n_hidden)]),
        fc2_w=sd["fc2.weight"].reshape(-1), fc2_b=sd["fc2.bias"].reshape(-1))


class RuntimePredictor:
    """mlp.py:112-146, 252-267: same constructor, attributes and predict().

    precision: "bf16", "bf16x3" (batched.MLPHandle) or "int8" (batched.Int8MLPHandle)."""

    def __init__(self, model_name, layers, layer_size, model_path=None, precision="bf16"):
        self.model_name = model_name
        self.layers = layers
        self.layer_size = layer_size
        self.model = _MODEL_CLASSES[model_name](layers, layer_size)
        self.device_params = ["mem", "mem_bw", "num_sm", "single"]
        self.mu = None
        self.sigma = None
        self.precision = precision
        self._handle = None
        self._device_rows = None
        self._momentum = None
        self._unchecked = None               # (GPU, dense.failures()) from before updates whose launches may have given up
        self._given_up = False               # one of them has
        if model_path is not None:
            self.load_state(model_path)

    # -- checkpoints --------------------------------------------------------
    def load_state(self, path):
        # mu / sigma are numpy arrays inside the checkpoint, which torch >= 2.6
        # only unpickles with weights_only=False
        checkpoint = torch.load(path, map_location="cpu", weights_only=False)
        self.mu = checkpoint["mu"]
        self.sigma = checkpoint["sigma"]
        self.model.load_state_dict(checkpoint["model"])
        self._momentum = self._unchecked = None
        self.invalidate()

    def save_state(self, path):
        self._check_updates()
        torch.save({"mu": self.mu, "sigma": self.sigma, "model": self.model.state_dict()}, path)

    def invalidate(self):
        """Drops the device-side weight pack (call after changing weights, mu or sigma).  A prediction that another
        thread is making keeps it until it has ended."""
        self._given_up = False
        self._handle = None
        self._device_rows = None

    # -- retraining ---------------------------------------------------------
    def update_hidden(self, lr, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5):
        """Steps the hidden layers' weights along orthogonalised updates, from the gradients that a backward pass has left in
        `model` (on a GPU, in float32; the reference's training loop does that with mlp.py:148-250): with g the gradients
        and m the kept momentum, m <- momentum m + g, the update is g + momentum m (nesterov) or m, made nearly orthogonal
        by `steps` Newton-Schulz steps (dense.orthogonalize, all layers in one call), and
        w <- (1 - lr weight_decay) w - lr update.  Biases, fc1 and fc2 are left to the caller's optimizer.
        The next prediction packs the new weights (`invalidate`).  Does not synchronise: whether a launch gave up on a bounded
        device wait, which leaves weights that mean nothing, is seen before they are packed or saved, and raised until they are
        replaced (`load_state`, or `invalidate` behind weights of the caller's)."""
        from habitat_b200 import dense
        weights = [block.weight for block in self.model.mlp.layers if isinstance(block, nn.Linear)]
        if any(w.grad is None for w in weights):
            raise RuntimeError("update_hidden needs the gradients of all hidden layers (run a backward pass first)")
        if any(not w.is_cuda or w.dtype != torch.float32 for w in weights):
            raise RuntimeError("update_hidden needs the model on a GPU, in float32")
        with torch.no_grad():
            g = torch.stack([w.grad for w in weights])
            kept = self._momentum
            if kept is None or kept.shape != g.shape or kept.device != g.device:
                kept = torch.zeros_like(g)
            kept = kept.mul(momentum).add_(g)
            update = torch.add(g, kept, alpha=momentum) if nesterov else kept
            if self._given_up or (self._unchecked is not None and self._unchecked[0] != g.device):
                self._check_updates()
            if self._unchecked is None:
                with torch.cuda.device(g.device):
                    unchecked = g.device, dense.failures()
            else:
                unchecked = self._unchecked
            step = dense.orthogonalize(update, steps=steps)       # what this raises leaves weights and momentum as they were
            if weight_decay:
                torch._foreach_mul_(weights, 1.0 - lr * weight_decay)
            torch._foreach_add_(weights, list(step.unbind(0)), alpha=-lr)
        self._momentum, self._unchecked = kept, unchecked
        self.invalidate()

    def _check_updates(self):
        from habitat_b200 import _native, dense
        if self._unchecked is not None:
            (device, since), self._unchecked = self._unchecked, None
            try:
                with torch.cuda.device(device):
                    dense.check_since(since)
            except _native.HabitatNativeError as e:
                if e.status != _native.HB_ERR_DEVICE_TIMEOUT:
                    raise
                self._given_up = True
        if self._given_up:
            raise _native.HabitatNativeError(_native.HB_ERR_DEVICE_TIMEOUT,
                                             "an update of the hidden layers gave up on a bounded wait: their weights mean nothing")

    # -- inference ----------------------------------------------------------
    def _ensure_handle(self):
        if self._handle is not None:
            return
        from habitat_b200.batched import Int8MLPHandle, MLPHandle
        if self.mu is None or self.sigma is None:
            raise RuntimeError("RuntimePredictor has no mu/sigma (load a checkpoint first)")
        self._check_updates()
        devices = get_all_devices(self.device_params)
        names = sorted(devices)
        self._device_rows = {name: i for i, name in enumerate(names)}
        table = np.array([devices[n] for n in names], dtype=np.float64)
        arrays = state_to_arrays(self.model)
        made = Int8MLPHandle if self.precision == "int8" else functools.partial(MLPHandle, precision=self.precision)
        self._handle = made(len(self.model.features), mu=np.asarray(self.mu, np.float64),
                            sigma=np.asarray(self.sigma, np.float64), device_features=table, **arrays)

    def device_row(self, device_name):
        self._ensure_handle()
        if device_name not in self._device_rows:
            get_device_features(device_name, self.device_params)  # raises like the reference
            self.invalidate()
            self._ensure_handle()
        return self._device_rows[device_name]

    def predict_batch(self, op_features, device_rows):
        """op_features [Q, F] float32 CUDA tensor, device_rows [Q] uint8 CUDA tensor
        (indices from device_row()).  Returns [Q] float32 predictions (ms), on the
        current stream, unsynchronised."""
        self._ensure_handle()
        return self._handle.predict(op_features, device_rows)

    def predict(self, kernel_arguments, device_name):
        """One query; same arguments and return type as the reference."""
        row = self.device_row(device_name)
        return self._handle.predict_one(kernel_arguments, row)
