"""Dense operators for the predictors' layers and their retraining: what is measured, and the plain forms.

* linear: rows quantised to 8-bit integers, one scale per row (token), times 8-bit weights with one scale per output
  channel, bias and ReLU (habitat_b200.dense.quantize_rows, int8_matmul);
* stack: several such layers, each handing 8-bit rows to the next one (int8_matmul_quantized in between);
* orthogonalize: the update of a weight matrix made nearly orthogonal by Newton-Schulz steps (orthogonalize).

Definition of the 8-bit rows, in float32 arithmetic: amax the row's largest magnitude, q = rint(x * (127 / amax)) with
ties to even, scale = amax / 127.  A product's value is (sum of the integer products as float32 * channel scale) * row
scale + bias, each operation rounded to float32, then ReLU.
"""
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7

#: The largest cases' multiplications: 8192^3 for one layer, and the stack's 65,536 rows through eight 1024-wide layers.
LINEAR_MOST = 8192 ** 3
STACK_MOST = 65536 * 1024 * 1024 * 8
ORTHOGONAL_MOST = 4096 * 4096 * 8192


def listed():
    return [
        # one query through one hidden layer of a predictor: latency
        {"name": "linear_1_query", "op": "linear", "m": 1, "n": 1024, "k": 1024, "dtype": "f32", "out": "f32", "bias": True, "relu": True},
        # a few tokens through a wide layer: the weights' bytes
        {"name": "linear_8_tokens_wide", "op": "linear", "m": 8, "n": 8192, "k": 8192, "dtype": "bf16", "out": "bf16", "bias": False, "relu": False},
        # odd sizes: a trace's 333 kernels, features and channels that end inside tiles
        {"name": "linear_odd", "op": "linear", "m": 333, "n": 1003, "k": 777, "dtype": "f16", "out": "f32", "bias": True, "relu": False},
        # the benchmark's 65,536 queries through one hidden layer
        {"name": "linear_65536_queries", "op": "linear", "m": 65536, "n": 1024, "k": 1024, "dtype": "bf16", "out": "bf16", "bias": True, "relu": True},
        # the largest product
        {"name": "linear_8192_cube", "op": "linear", "m": 8192, "n": 8192, "k": 8192, "dtype": "bf16", "out": "bf16", "bias": False, "relu": False},
        # a small batch of queries through a predictor's eight hidden layers
        {"name": "stack_127_queries", "op": "stack", "m": 127, "width": 1024, "layers": 8, "dtype": "f32", "out": "f32"},
        # a middle batch through narrower layers
        {"name": "stack_4096_narrow", "op": "stack", "m": 4096, "width": 500, "layers": 4, "dtype": "bf16", "out": "bf16"},
        # the benchmark's batch through a predictor's eight hidden layers
        {"name": "stack_65536_queries", "op": "stack", "m": 65536, "width": 1024, "layers": 8, "dtype": "f32", "out": "bf16"},
        # the update of a predictor's first layer (conv2d: 8 features and 4 of the device)
        {"name": "orthogonalize_first_layer", "op": "orthogonalize", "batch": 1, "rows": 1024, "cols": 12, "dtype": "f32"},
        # the updates of a predictor's eight hidden layers at a time
        {"name": "orthogonalize_hidden", "op": "orthogonalize", "batch": 8, "rows": 1024, "cols": 1024, "dtype": "f32"},
        # an odd matrix in 16 bits
        {"name": "orthogonalize_odd", "op": "orthogonalize", "batch": 1, "rows": 1000, "cols": 777, "dtype": "f16"},
        # a large layer's update in 16 bits
        {"name": "orthogonalize_large", "op": "orthogonalize", "batch": 1, "rows": 8192, "cols": 4096, "dtype": "bf16"},
    ]


def _spread(rng, low, high):
    """A whole number, spread over the logarithm of the range."""
    return min(high, max(low, int(low * (high / low) ** rng.random() + 0.5)))


def draw(rng):
    op = rng.choice(["linear", "linear", "stack", "orthogonalize", "orthogonalize"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "linear":
        while True:
            m, n, k = _spread(rng, 1, 65536), _spread(rng, 1, 8192), _spread(rng, 1, 8192)
            if m * n * k <= LINEAR_MOST and m * max(n, k) <= 2 ** 27:
                return {"op": op, "m": m, "n": n, "k": k, "dtype": dtype, "out": rng.choice(["f32", "bf16", "f16"]),
                        "bias": rng.random() < 0.5, "relu": rng.random() < 0.5}
    if op == "stack":
        while True:
            m, width, layers = _spread(rng, 1, 65536), _spread(rng, 16, 1024), rng.randint(2, 8)
            if m * width * width * layers <= STACK_MOST:
                return {"op": op, "m": m, "width": width, "layers": layers, "dtype": dtype,
                        "out": rng.choice(["f32", "bf16", "f16"])}
    while True:
        batch, rows, cols = rng.choice([1, 1, 2, 5, 8]), _spread(rng, 1, 8192), _spread(rng, 1, 8192)
        if batch * min(rows, cols) ** 2 * max(rows, cols) <= ORTHOGONAL_MOST and batch * rows * cols <= 2 ** 26:
            return {"op": op, "batch": batch, "rows": rows, "cols": cols, "dtype": dtype}


def _weights(g, n, k):
    """A trained layer's weights in 8 bits with a scale per output channel, channels of different sizes."""
    w = torch.randn((n, k), generator=g, device="cuda") * torch.exp(0.3 * torch.randn((n, 1), generator=g, device="cuda"))
    w *= (2.0 / k) ** 0.5
    scale = w.abs().amax(dim=1).clamp_min(1e-12) / 127.0
    return torch.round(w / scale[:, None]).clamp_(-127, 127).to(torch.int8), scale


def _activations(g, m, k, dtype):
    """Rows as they come out of a ReLU (half of them zeros) or as they enter a network, with sizes that differ from row to row."""
    x = torch.randn((m, k), generator=g, device="cuda")
    x[: m // 2].clamp_min_(0.0)
    x *= torch.exp(torch.randn((m, 1), generator=g, device="cuda"))
    return x.to(DTYPES[dtype])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if case["op"] == "linear":
        state["x"] = _activations(g, case["m"], case["k"], case["dtype"])
        state["weight"], state["scale"] = _weights(g, case["n"], case["k"])
        state["bias"] = 0.1 * torch.randn((case["n"],), generator=g, device="cuda") if case["bias"] else None
    elif case["op"] == "stack":
        state["x"] = _activations(g, case["m"], case["width"], case["dtype"])
        state["layers"] = []
        for _ in range(case["layers"]):
            weight, scale = _weights(g, case["width"], case["width"])
            state["layers"].append((weight, scale, 0.1 * torch.randn((case["width"],), generator=g, device="cuda")))
    else:
        # a momentum: a few strong directions over the noise of many batches
        b, r, c = case["batch"], case["rows"], case["cols"]
        strong = max(1, min(r, c) // 16)
        u = torch.randn((b, r, strong), generator=g, device="cuda")
        v = torch.randn((b, strong, c), generator=g, device="cuda")
        noise = torch.randn((b, r, c), generator=g, device="cuda")
        state["update"] = (1e-3 * (torch.matmul(u, v) * strong ** -0.5 + noise)).to(DTYPES[case["dtype"]])
    return state


# -- plain forms ------------------------------------------------------------

def _quantize_rows(x):
    x = x.float()
    amax = x.abs().amax(dim=1)
    # tensor by tensor: a division with a Python number goes through its reciprocal, which rounds twice
    most = torch.full_like(amax, 127.0)
    inverse = torch.where(amax > 0, most / amax, torch.zeros_like(amax))
    return torch.round(x * inverse[:, None]), amax / most


def _product(q, q_scale, weight, scale, bias, relu):
    # the sums of whole numbers are exact in float32 up to 2^24, in float64 beyond
    wide = torch.float32 if q.shape[1] * 127 * 127 < 2 ** 24 else torch.float64
    sums = torch.matmul(q.to(wide), weight.to(wide).t()).float()
    y = sums * scale * q_scale[:, None]
    if bias is not None:
        y = y + bias
    return torch.relu(y) if relu else y


def _newton_schulz(update, steps=5):
    x = update.float()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1)
    a, b, c = COEFFICIENTS
    x = x / ((x * x).sum(dim=(-2, -1), keepdim=True).sqrt() + EPS)
    for _ in range(steps):
        gram = torch.matmul(x, x.transpose(-2, -1))
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return (x.transpose(-2, -1) if tall else x).to(update.dtype).contiguous()


def run(state):
    case = state["case"]
    if own:
        from habitat_b200 import dense
        if case["op"] == "linear":
            q, q_scale = dense.quantize_rows(state["x"])
            return dense.int8_matmul(q, q_scale, state["weight"], state["scale"], bias=state["bias"], relu=case["relu"],
                                     out_dtype=DTYPES[case["out"]])
        if case["op"] == "stack":
            q, q_scale = dense.quantize_rows(state["x"])
            for weight, scale, bias in state["layers"][:-1]:
                q, q_scale = dense.int8_matmul_quantized(q, q_scale, weight, scale, bias=bias, relu=True)
            weight, scale, bias = state["layers"][-1]
            return dense.int8_matmul(q, q_scale, weight, scale, bias=bias, relu=True, out_dtype=DTYPES[case["out"]])
        return dense.orthogonalize(state["update"], steps=5, coefficients=COEFFICIENTS, eps=EPS)
    if case["op"] == "linear":
        q, q_scale = _quantize_rows(state["x"])
        return _product(q, q_scale, state["weight"], state["scale"], state["bias"], case["relu"]).to(DTYPES[case["out"]])
    if case["op"] == "stack":
        y = state["x"]
        for weight, scale, bias in state["layers"]:
            q, q_scale = _quantize_rows(y)
            y = _product(q, q_scale, weight, scale, bias, True)
        return y.to(DTYPES[case["out"]])
    return _newton_schulz(state["update"])


def work(case):
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k * SIZES[case["dtype"]] + n * k + 4 * n * (2 if case["bias"] else 1) + m * n * SIZES[case["out"]],
                "flops": 2 * m * n * k}
    if case["op"] == "stack":
        m, w, layers = case["m"], case["width"], case["layers"]
        return {"bytes": m * w * (SIZES[case["dtype"]] + SIZES[case["out"]]) + layers * (w * w + 8 * w),
                "flops": 2 * m * w * w * layers}
    # of the two symmetric products of a step half has to be computed
    s, l = sorted((case["rows"], case["cols"]))
    return {"bytes": 2 * case["batch"] * s * l * SIZES[case["dtype"]],
            "flops": case["batch"] * 5 * (s * s * l + s * s * s + 2 * s * s * l)}


# -- in 64 bits -------------------------------------------------------------

def _as_float32(x):
    """Rounds float64 values where the definition has a float32 value."""
    return x.to(torch.float32).to(torch.float64)


def _layer_in_64_bits(x, weight, scale, bias, relu):
    """One layer on float64 rows whose values are float32 numbers; the definition's roundings and no others."""
    largest = x.abs().max(dim=1, keepdim=True).values
    whole = torch.round(_as_float32(x * _as_float32(127.0 / largest.clamp_min(1e-30))))   # rows of zeros stay so
    acc = _as_float32(whole @ weight.double().T)
    y = _as_float32(_as_float32(acc * scale.double()) * _as_float32(largest / 127.0))
    if bias is not None:
        y = y + bias.double()
    return y.clamp_min(0.0) if relu else y


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "linear":
        return _layer_in_64_bits(state["x"].double(), state["weight"], state["scale"], state["bias"], case["relu"])
    if case["op"] == "stack":
        y = state["x"].double()
        for weight, scale, bias in state["layers"]:
            y = _as_float32(_layer_in_64_bits(y, weight, scale, bias, True))
        return y
    x = state["update"].double()
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + EPS)
    flip = case["rows"] > case["cols"]
    a, b, c = COEFFICIENTS
    eye = torch.eye(min(case["rows"], case["cols"]), dtype=torch.float64, device=x.device)
    for _ in range(5):
        gram = x.mT @ x if flip else x @ x.mT
        factor = a * eye + b * gram + c * (gram @ gram)
        x = x @ factor if flip else factor @ x
    return x
