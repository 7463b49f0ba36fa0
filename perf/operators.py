"""What is timed of the training operators: updates of the primitives' and the decoder's weight matrices by their
orthogonalised momentum, and the way of rows from pixels to the primitives that their records name and back.

    orthogonalize   muon.orthogonalize: Newton-Schulz iteration on a stack of matrices
    muon            muon.muon_step: momentum, orthogonalisation and weight update, in place
    route           primitive_csr.route_records: the place of every record among the records grouped by primitive
    dispatch        primitive_csr.dispatch_rows (forward) and dispatch_rows_gradient: a pixel's row to each of its records
    combine         primitive_csr.combine_rows (forward) and combine_rows_gradients: weighted sum of a pixel's records

Records come in two layouts: `fan` records for every pixel (a router's choice of experts, some of them dropped), and
lists of any length per pixel (the records of a rendered image; fan = 0, about `hits` of them a pixel).
"""
import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS, EPS = 5, 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # the decoder's 3x3 convolution as one matrix: a single update, all latency
        dict(name="orthogonalize_128x1152", kind="orthogonalize", n=1, rows=128, cols=1152, dtype="fp32"),
        # first layers of a middling scene, an odd count, in bfloat16
        dict(name="orthogonalize_20001x32x72", kind="orthogonalize", n=20_001, rows=32, cols=72, dtype="bf16"),
        # one step on the primitives of the smallest scene
        dict(name="muon_2k_hidden32", kind="muon", n=2_000, hidden=32, inputs=72, grads="fp32", masked=False),
        # the largest: one step on the primitives of the headline scene, 345 million weights
        dict(name="muon_100k_hidden32", kind="muon", n=100_000, hidden=32, inputs=72, grads="fp32", masked=False),
        # wide hidden layers, binary16 gradients, primitives that no record reached left alone
        dict(name="muon_15001_hidden64_masked", kind="muon", n=15_001, hidden=64, inputs=72, grads="fp16", masked=True),
        # one step on the feature decoder's three layers
        dict(name="muon_decoder_128_128_512", kind="muon_decoder", inputs=128, hidden=128, outputs=512, grads="fp32"),
        # a router's choice: four of 256 experts for each of 8,191 rows, one slot in twenty dropped
        dict(name="route_8191x4_of_256", kind="route", pixels=8_191, fan=4, primitives=256, hits=0.0),
        # the records of one 1200x680 image
        dict(name="route_image_100k_1200x680", kind="route", pixels=1200 * 680, fan=0, primitives=100_000, hits=9.5),
        # wide rows to their experts
        dict(name="dispatch_8191x4_512_bf16", kind="dispatch", pixels=8_191, fan=4, primitives=256, hits=0.0, dim=512,
             dtype="bf16", direction="forward"),
        # the gradient of a small image's features that were handed to its records
        dict(name="dispatch_gradient_320x240_128", kind="dispatch", pixels=320 * 240, fan=0, primitives=20_000, hits=9.5,
             dim=128, dtype="fp32", direction="gradient"),
        # a single row back from its eight experts: latency
        dict(name="combine_1x8_512_fp16", kind="combine", pixels=1, fan=8, primitives=64, hits=0.0, dim=512, dtype="fp16",
             direction="forward"),
        # colour and depth of an image from its records, with both gradients
        dict(name="combine_training_800x600_4", kind="combine", pixels=800 * 600, fan=0, primitives=50_000, hits=9.5, dim=4,
             dtype="fp32", direction="training"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["orthogonalize", "orthogonalize", "muon", "muon", "muon_decoder", "route", "dispatch", "dispatch", "combine",
                       "combine", "combine"])
    if kind == "orthogonalize":
        small = _log(rng, 1, 128)
        large = _log(rng, small, 2_048)
        rows, cols = rng.choice([(small, large), (large, small)])
        most = min(2.0e7 / (rows * cols), 4.0e10 / _newton_schulz_flops(1, rows, cols), 50_000.0)
        return dict(kind=kind, n=_log(rng, 1, max(1.0, most)), rows=rows, cols=cols, dtype=rng.choice(list(TYPES)))
    if kind == "muon":
        hidden, inputs = rng.choice([8, 16, 24, 32, 32, 32, 48, 64]), 12 * rng.randint(3, 8)
        most = 8.0e7 / (hidden * (inputs + hidden + 4))
        return dict(kind=kind, n=_log(rng, 500, min(most, 40_000)), hidden=hidden, inputs=inputs, grads=rng.choice(list(TYPES)),
                    masked=rng.random() < 0.4)
    if kind == "muon_decoder":
        return dict(kind=kind, inputs=_log(rng, 16, 128), hidden=rng.choice([32, 64, 96, 128]), outputs=_log(rng, 64, 768),
                    grads=rng.choice(list(TYPES)))
    c = dict(kind=kind)
    if rng.random() < 0.5:
        c.update(fan=rng.choice([1, 2, 3, 4, 6, 8]), hits=0.0, primitives=_log(rng, 4, 4_096))
        c["pixels"] = _log(rng, 1, 400_000 // c["fan"])
    else:
        c.update(fan=0, hits=round(rng.uniform(1.0, 16.0), 2), primitives=_log(rng, 500, 400_000))
        c["pixels"] = _log(rng, 64, 3.0e6 / c["hits"])
    if kind == "route":
        return c
    records = c["pixels"] * (c["fan"] or c["hits"])
    c["dim"] = _log(rng, 1, max(1.0, min(1_024.0, 8.0e7 / records)))
    c["dtype"] = rng.choice(list(TYPES))
    c["direction"] = rng.choice(["forward", "gradient"] if kind == "dispatch" else ["forward", "training"])
    return c


# ---------------------------------------------------------------------------------------------------------- inputs ----
def _gradients(g, n, rows, cols, dtype, empty=0.0):
    """Sums over many records: a dominant direction over a full-rank rest, their size differing between matrices by
    orders of magnitude; a share `empty` of the matrices saw no record."""
    x = torch.randn(n, rows, cols, generator=g, device="cuda")
    x += 1.5 * torch.randn(n, rows, 1, generator=g, device="cuda") * torch.randn(n, 1, cols, generator=g, device="cuda")
    x *= torch.exp(torch.randn(n, 1, 1, generator=g, device="cuda") - 5.0)
    if empty > 0.0:
        x *= (torch.rand(n, 1, 1, generator=g, device="cuda") >= empty)
    return x.to(TYPES[dtype])


def _layers(case):
    if case["kind"] == "muon_decoder":
        return [(1, case["hidden"], case["inputs"]), (1, case["hidden"], 9 * case["hidden"]), (1, case["outputs"], case["hidden"])]
    return [(case["n"], case["hidden"], case["inputs"]), (case["n"], case["hidden"], case["hidden"]), (case["n"], 4, case["hidden"])]


def _record_ids(case, g):
    """(ids, first record of every pixel or None).  An image's records: the pixels of a strip of 64 share a list of
    primitives, from which each takes a run; a router's: skewed choices, one in twenty dropped."""
    T, N, fan = case["pixels"], case["primitives"], case["fan"]
    if fan:
        ids = (N * torch.rand(T, fan, generator=g, device="cuda") ** 1.5).to(torch.int32).clamp_(max=N - 1)
        return torch.where(torch.rand(T, fan, generator=g, device="cuda") < 0.05, torch.full_like(ids, -1), ids), None
    counts = torch.randperm(T, generator=g, device="cuda") % (int(2 * case["hits"]) + 1)      # their sum is the case's
    first = torch.zeros(T + 1, dtype=torch.int64, device="cuda")
    torch.cumsum(counts, 0, out=first[1:])
    lists = torch.randint(0, N, ((T + 63) // 64, 48), generator=g, device="cuda", dtype=torch.int32)
    pixel = torch.repeat_interleave(torch.arange(T, device="cuda"), counts)
    start = torch.randint(0, 16, (T,), generator=g, device="cuda")
    place = start[pixel] + torch.arange(pixel.numel(), device="cuda") - first[pixel]
    return lists[pixel // 64, place % 48], first


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = dict(case=case)
    if case["kind"] == "orthogonalize":
        s["update"] = _gradients(g, case["n"], case["rows"], case["cols"], case["dtype"])
        if case["n"] == 1:
            s["update"] = s["update"][0]
        return s
    if case["kind"] in ("muon", "muon_decoder"):
        layers, empty = _layers(case), 0.1 if case["kind"] == "muon" else 0.0
        s["weights"] = [torch.randn(*shape, generator=g, device="cuda") / math.sqrt(shape[2]) for shape in layers]
        s["grads"] = [_gradients(g, *shape, case["grads"], empty) for shape in layers]
        s["momenta"] = [0.3 * _gradients(g, *shape, "fp32") for shape in layers]
        s["active"] = torch.rand(case["n"], generator=g, device="cuda") < 0.7 if case.get("masked") else None
        if case["kind"] == "muon_decoder":
            for k in ("weights", "grads", "momenta"):
                s[k] = [t[0] for t in s[k]]
        return s
    s["ids"], s["first"] = _record_ids(case, g)
    if case["kind"] == "route":
        return s
    N, R = case["primitives"], s["ids"].numel()
    key = torch.where(s["ids"] < 0, N, s["ids"]).reshape(-1)
    order = torch.sort(key, stable=True)[1]
    s["slots"] = torch.empty(R, dtype=torch.int32, device="cuda")
    s["slots"][order] = torch.arange(R, dtype=torch.int32, device="cuda")
    s["offsets"] = torch.zeros(N + 1, dtype=torch.int64, device="cuda")
    s["offsets"][1:] = torch.cumsum(torch.bincount(key, minlength=N + 1)[:N], 0)
    dtype, D, T = TYPES[case["dtype"]], case["dim"], case["pixels"]
    if case["kind"] == "dispatch":
        rows = T if case["direction"] == "forward" else R
        s["x"] = torch.randn(rows, D, generator=g, device="cuda").to(dtype)
        return s
    s["y"] = torch.randn(R, D, generator=g, device="cuda").to(dtype)
    s["weights"] = torch.rand(s["ids"].shape, generator=g, device="cuda")
    s["grad"] = torch.randn(T, D, generator=g, device="cuda").to(dtype) if case["direction"] == "training" else None
    return s


# -------------------------------------------------------------------------------------------------- one pass: plain ----
def _newton_schulz(u):
    """`u` [n, rows, cols] in 32 bits."""
    a, b, c = COEFFICIENTS
    tall = u.shape[1] > u.shape[2]
    x = u.transpose(1, 2) if tall else u
    x = x / x.square().sum((1, 2), keepdim=True).sqrt().clamp(min=EPS)
    for _ in range(STEPS):
        gram = x @ x.transpose(1, 2)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(1, 2) if tall else x


def _stack(t):
    return t if t.dim() == 3 else t[None]


def _plain_muon(s):
    for w, grad, m in zip(s["weights"], s["grads"], s["momenta"]):
        w, grad, m = _stack(w), _stack(grad).float(), _stack(m)
        on = slice(None) if s["active"] is None else s["active"].nonzero()[:, 0]
        grad = grad[on]
        new = m[on] + (1.0 - MOMENTUM) * (grad - m[on])
        update = _newton_schulz(grad + MOMENTUM * (new - grad))
        scale = LR * math.sqrt(max(1.0, w.shape[1] / w.shape[2]))
        w[on] = w[on] * (1.0 - LR * DECAY) - scale * update
        m[on] = new
    return dict(weights=s["weights"], momenta=s["momenta"])


def _plain_route(s):
    ids, N = s["ids"].reshape(-1), s["case"]["primitives"]
    key = torch.where((ids < 0) | (ids >= N), N, ids)
    order = torch.sort(key, stable=True)[1]
    slots = torch.empty(ids.numel(), dtype=torch.int32, device=ids.device)
    slots[order] = torch.arange(ids.numel(), dtype=torch.int32, device=ids.device)
    offsets = torch.zeros(N + 1, dtype=torch.int64, device=ids.device)
    offsets[1:] = torch.cumsum(torch.bincount(key, minlength=N + 1)[:N], 0)
    return dict(offsets=offsets, slots=slots)


def _pixels(s):
    """The pixel of every record."""
    T, fan = s["case"]["pixels"], s["case"]["fan"]
    every = torch.arange(T, device=s["slots"].device)
    return every.repeat_interleave(fan if fan else s["first"][1:] - s["first"][:-1], output_size=s["slots"].numel())


def _sum_records(s, rows):
    """Sums of the records' rows [R, D] per pixel."""
    T, fan = s["case"]["pixels"], s["case"]["fan"]
    if fan:
        return rows.view(T, fan, -1).sum(1)
    return torch.zeros(T, rows.shape[1], device=rows.device).index_add_(0, _pixels(s), rows)


def _plain_dispatch(s):
    slots, x = s["slots"].long(), s["x"]
    kept = (slots < s["offsets"][-1])[:, None]
    if s["case"]["direction"] == "forward":
        out = torch.empty(slots.numel(), x.shape[1], dtype=x.dtype, device=x.device)
        out[slots] = torch.where(kept, x[_pixels(s)], 0)
        return out
    return _sum_records(s, torch.where(kept, x[slots].float(), 0.0)).to(x.dtype)


def _plain_combine(s):
    slots, y, weights = s["slots"].long(), s["y"], s["weights"].reshape(-1, 1)
    kept = (slots < s["offsets"][-1])[:, None]
    rows = torch.where(kept, y[slots].float(), 0.0)
    out = dict(out=_sum_records(s, weights * rows).to(y.dtype))
    if s["case"]["direction"] == "training":
        grad = s["grad"].float()[_pixels(s)]
        grad_y = torch.empty_like(y)
        grad_y[slots] = torch.where(kept, weights * grad, 0.0).to(y.dtype)
        out.update(grad_y=grad_y, grad_weights=(rows * grad).sum(1).view(s["weights"].shape))
    return out


# ---------------------------------------------------------------------------------------------- one pass: framework ----
def _route(s):
    from mlp_splatting_b200.primitive_csr import RecordRoute
    return RecordRoute(s["offsets"], s["slots"], s["case"]["pixels"], s["case"]["fan"], s["first"])


def _run_own(s):
    from mlp_splatting_b200 import muon, primitive_csr
    kind = s["case"]["kind"]
    if kind == "orthogonalize":
        return muon.orthogonalize(s["update"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
    if kind in ("muon", "muon_decoder"):
        muon.muon_step(s["weights"], s["grads"], s["momenta"], lr=LR, momentum=MOMENTUM, weight_decay=DECAY, steps=STEPS,
                       coefficients=COEFFICIENTS, eps=EPS, active=s["active"])
        return dict(weights=s["weights"], momenta=s["momenta"])
    if kind == "route":
        route = primitive_csr.route_records(s["ids"], s["case"]["primitives"], s["first"])
        return dict(offsets=route.offsets, slots=route.slots)
    if kind == "dispatch":
        if s["case"]["direction"] == "forward":
            return primitive_csr.dispatch_rows(s["x"], _route(s))
        return primitive_csr.dispatch_rows_gradient(s["x"], _route(s))
    route = _route(s)
    out = dict(out=primitive_csr.combine_rows(s["y"], route, s["weights"]))
    if s["case"]["direction"] == "training":
        out["grad_y"], out["grad_weights"] = primitive_csr.combine_rows_gradients(s["grad"], s["y"], route, s["weights"])
    return out


def run(s):
    if own:
        return _run_own(s)
    kind = s["case"]["kind"]
    if kind == "orthogonalize":
        return _newton_schulz(_stack(s["update"]).float()).to(s["update"].dtype).view(s["update"].shape)
    if kind in ("muon", "muon_decoder"):
        return _plain_muon(s)
    return {"route": _plain_route, "dispatch": _plain_dispatch, "combine": _plain_combine}[kind](s)


# ------------------------------------------------------------------------------------------------------------- work ----
def _newton_schulz_flops(n, rows, cols):
    small, large = min(rows, cols), max(rows, cols)
    return STEPS * n * (4.0 * small * small * large + 2.0 * small ** 3)


def work(case):
    kind = case["kind"]
    if kind == "orthogonalize":
        size = 4 if case["dtype"] == "fp32" else 2
        return dict(bytes=2 * size * case["n"] * case["rows"] * case["cols"],
                    flops=_newton_schulz_flops(case["n"], case["rows"], case["cols"]))
    if kind in ("muon", "muon_decoder"):
        share = 0.7 if case.get("masked") else 1.0      # of the primitives whose matrices are touched
        each = 16 + (4 if case["grads"] == "fp32" else 2)      # gradient read; momentum and weight read and written
        return dict(bytes=share * sum(each * n * r * c for n, r, c in _layers(case)),
                    flops=share * sum(_newton_schulz_flops(*shape) for shape in _layers(case)))
    T, N = case["pixels"], case["primitives"]
    lengths = int(2 * case["hits"]) + 1
    R = T * case["fan"] or T // lengths * (lengths * (lengths - 1) // 2) + T % lengths * (T % lengths - 1) // 2
    if kind == "route":
        return dict(bytes=8 * R + 8 * (N + 1), flops=0)
    index = 4 * R + (0 if case["fan"] else 8 * (T + 1))
    size = 4 if case["dtype"] == "fp32" else 2
    rows = size * case["dim"] * (R + T)
    if kind == "dispatch":
        return dict(bytes=index + rows, flops=0 if case["direction"] == "forward" else R * case["dim"])
    if case["direction"] == "forward":
        return dict(bytes=index + 4 * R + rows, flops=2 * R * case["dim"])
    # once each: records' rows, weights, incoming gradient, output; both gradients written
    return dict(bytes=index + 4 * R + rows + size * case["dim"] * T + size * case["dim"] * R + 4 * R, flops=5 * R * case["dim"])


# ------------------------------------------------------------------------------------------------- from 64 bits ----
def _exact_polar(u):
    """Newton-Schulz iteration on the smaller Gram side, in 64 bits, some thousand matrices at a time."""
    out = torch.empty(u.shape, dtype=torch.float64, device=u.device)
    p, q, r = COEFFICIENTS
    for i in range(0, u.shape[0], 8_192):
        x = u[i:i + 8_192].double()
        x = x / torch.linalg.vector_norm(x, dim=(1, 2), keepdim=True).clamp(min=EPS)
        for _ in range(STEPS):
            if x.shape[1] <= x.shape[2]:
                s = torch.bmm(x, x.mT)
                x = p * x + torch.bmm(q * s + r * torch.bmm(s, s), x)
            else:
                s = torch.bmm(x.mT, x)
                x = p * x + torch.bmm(x, q * s + r * torch.bmm(s, s))
        out[i:i + 8_192] = x
    return out


def _exact_muon(s):
    weights, momenta = [], []
    for w, grad, m in zip(s["weights"], s["grads"], s["momenta"]):
        shape, w, grad, m = w.shape, _stack(w).double(), _stack(grad).double(), _stack(m).double()
        new = MOMENTUM * m + (1.0 - MOMENTUM) * grad
        step = _exact_polar((1.0 - MOMENTUM) * grad + MOMENTUM * new) * math.sqrt(max(1.0, w.shape[1] / w.shape[2]))
        after = w - LR * (DECAY * w + step)
        if s["active"] is not None:
            off = ~s["active"]
            new[off], after[off] = m[off], w[off]
        weights.append(after.view(shape))
        momenta.append(new.view(shape))
    return dict(weights=weights, momenta=momenta)


def exact(case, seed):
    if case["kind"] == "route":
        return None
    s = prepare(case, seed)
    if case["kind"] == "orthogonalize":
        return _exact_polar(_stack(s["update"])).view(s["update"].shape)
    if case["kind"] in ("muon", "muon_decoder"):
        return _exact_muon(s)
    T, fan, D = case["pixels"], case["fan"], case["dim"]
    kept, slots = int(s["offsets"][-1]), s["slots"].long()
    first = s["first"] if s["first"] is not None else fan * torch.arange(T + 1, device="cuda")
    pixel = torch.bucketize(torch.arange(slots.numel(), device="cuda"), first[1:], right=True)
    if case["kind"] == "dispatch" and case["direction"] == "forward":
        order = torch.argsort(slots)
        out = s["x"].double()[pixel[order]]
        out[kept:] = 0.0
        return out

    def per_pixel(rows):
        run = torch.cat([rows.new_zeros(1, D), torch.cumsum(rows, 0)])
        return run[first[1:]] - run[first[:-1]]

    if case["kind"] == "dispatch":
        rows = s["x"].double()
        rows[kept:] = 0.0
        return per_pixel(rows[slots])
    rows, weights = s["y"].double(), s["weights"].double().reshape(-1)
    rows[kept:] = 0.0
    out = dict(out=per_pixel(weights[:, None] * rows[slots]))
    if case["direction"] == "training":
        order = torch.argsort(slots)
        grad = s["grad"].double()
        grad_y = weights[order][:, None] * grad[pixel[order]]
        grad_y[kept:] = 0.0
        out.update(grad_y=grad_y, grad_weights=torch.einsum("rd,rd->r", rows[slots], grad[pixel]).view(s["weights"].shape))
    return out
