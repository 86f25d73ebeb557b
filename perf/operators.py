"""What is timed of the classifier loss and of the orthogonalised update, and their plain forms.

Operators (include/mi_mlp.h):
  xent_forward   loss_i = lse_i - z_i[t_i], lse_i = log sum_j exp z_ij, z = X W^T + b, without keeping z
  xent_backward  g_ij = d_i (exp(z_ij - lse_i) - [j = t_i]);  dX = g W, dW = g^T X, db = column sums of g
  orthogonalize  O = X_s of  X <- a X + (b A + c A^2) X, A = X X^T, from X_0 = G / |G|_F
  ortho_update   momentum over the summed replicas, O of it, W <- (1 - lr wd) W - lr scale O, bf16 copies W and W^T

With `own` false, run() computes them with elementary torch operations in 32 bits; with `own` true it
makes the calls of the C ABI that a user makes."""
import math

import torch

own = False

COEF = (3.4445, -4.7750, 2.0315)
MUON_STEPS = 5


# ---- cases ---------------------------------------------------------------------------------------

def _xent(op, name, dtype, rows, vocab, width, bias):
    return {"name": name, "op": op, "dtype": dtype, "rows": rows, "vocab": vocab, "width": width, "bias": bias}


def listed():
    return [
        # the score of one token: the weights are read once, the call's own latency counts
        _xent("xent_forward", "xent_fwd_one_token", "bf16", 1, 32000, 1024, False),
        # one micro-batch of an ordinary model, a vocabulary that is no multiple of anything, with a bias
        _xent("xent_forward", "xent_fwd_odd_vocab", "bf16", 4096, 50021, 2048, True),
        # the whole batch of the largest configuration (16384 rows) against a large vocabulary
        _xent("xent_forward", "xent_fwd_large", "bf16", 16384, 131072, 4096, False),
        # an fp32 model of the default width, one replica's batch
        _xent("xent_forward", "xent_fwd_f32", "f32", 1024, 32000, 1024, True),
        # a small classifier: a chain of short launches
        _xent("xent_backward", "xent_bwd_small", "bf16", 256, 1000, 512, True),
        _xent("xent_backward", "xent_bwd_odd_vocab", "bf16", 4096, 50021, 2048, True),
        _xent("xent_backward", "xent_bwd_large", "bf16", 8192, 131072, 4096, False),
        _xent("xent_backward", "xent_bwd_f32", "f32", 1024, 10007, 1024, True),
        # one layer of the smallest configuration (512 x 512), fp32 gradient
        {"name": "ortho_one_512", "op": "orthogonalize", "dtype": "f32", "batch": 1, "rows": 512, "cols": 512},
        # odd, tall, bf16 gradient
        {"name": "ortho_odd_tall", "op": "orthogonalize", "dtype": "bf16", "batch": 2, "rows": 4100, "cols": 1000},
        # all eight layers of the headline configuration in one call, four replicas
        {"name": "ortho_update_8x1024", "op": "ortho_update", "batch": 8, "rows": 1024, "cols": 1024, "replicas": 4},
        # one layer of the largest configuration, four replicas
        {"name": "ortho_update_8192", "op": "ortho_update", "batch": 1, "rows": 8192, "cols": 8192, "replicas": 4},
    ]


def _log(rng, lo, hi):
    """A size spread over its logarithm; one in two is odd or a little off a round number."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        v = max(lo, v // 64 * 64) if v >= 64 else v
    return min(hi, max(lo, v))


def draw(rng):
    op = rng.choice(["xent_forward", "xent_backward", "orthogonalize", "ortho_update"])
    if op.startswith("xent"):
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        most = {("xent_forward", "bf16"): 8.5e12, ("xent_backward", "bf16"): 4e12}.get((op, dtype), 1e10)
        rows, vocab, width = _log(rng, 1, 16384), _log(rng, 1000, 131072), _log(rng, 128, 4096)
        if rows * vocab * width > most:
            rows = max(1, int(most / (vocab * width)))
        return {"op": op, "dtype": dtype, "rows": rows, "vocab": vocab, "width": width, "bias": rng.random() < 0.5}
    rows, cols = _log(rng, 64, 8192), _log(rng, 64, 8192)
    batch = rng.randint(1, 8)
    while batch > 1 and batch * rows * cols > 8192 * 8192 // 4:
        batch -= 1
    if op == "orthogonalize":
        return {"op": op, "dtype": rng.choice(["f32", "bf16"]), "batch": batch, "rows": rows, "cols": cols}
    return {"op": op, "batch": batch, "rows": rows, "cols": cols, "replicas": rng.randint(1, 4)}


# ---- inputs --------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    op = case["op"]
    if op.startswith("xent"):
        M, V, K = case["rows"], case["vocab"], case["width"]
        dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        W = randn(V, K).mul_(2.5 / math.sqrt(K))
        target = torch.randint(0, V, (M,), generator=gen, device="cuda")
        # some rows know their answer, some do not
        X = randn(M, K) + 4.0 * torch.rand(M, 1, generator=gen, device="cuda") * W[target]
        ignored = torch.rand(M, generator=gen, device="cuda") < 0.1  # padding
        target[ignored] = -1
        if M == 1:
            target.clamp_(min=0)
        state = {"case": case, "X": X.to(dt), "W": W.to(dt), "bias": randn(V) if case["bias"] else None,
                 "target": target.to(torch.int32)}
        if op == "xent_backward":
            if dt == torch.bfloat16:
                state["Wt"] = state["W"].t().contiguous()  # the copy that the update of a bf16 model writes beside W
            lse = torch.empty(M, device="cuda")
            for i in range(0, M, 2048):  # what the forward call has left behind
                z = state["X"][i:i + 2048].float() @ state["W"].float().t()
                if state["bias"] is not None:
                    z += state["bias"]
                lse[i:i + 2048] = torch.logsumexp(z, 1)
            state["lse"] = lse
            valid = state["target"] >= 0
            state["dloss"] = valid.float() / valid.sum().clamp(min=1)  # of the mean over the rows that count
        return state
    b, m, n = case["batch"], case["rows"], case["cols"]
    # gradients of a layer: a few strong directions over a noise floor
    r = max(1, min(m, n) // 16)
    if op == "orthogonalize":
        G = randn(b, m, r) @ randn(b, r, n) / math.sqrt(r) + 0.3 * randn(b, m, n)
        return {"case": case, "G": (1e-3 * G).to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)}
    R = case["replicas"]
    common = randn(b, m, r) @ randn(b, r, n) / math.sqrt(r)
    G = torch.empty(R, b, m, n, device="cuda")
    for k in range(R):
        G[k] = 1e-3 / R * (common + 0.5 * randn(b, m, n))
    W = randn(b, m, n).mul_(1.0 / math.sqrt(n))
    return {"case": case, "G": G, "momentum": 1e-3 * (3.0 * common + randn(b, m, n)), "W": W,
            "W16": W.to(torch.bfloat16), "Wt16": W.transpose(1, 2).to(torch.bfloat16).contiguous(),
            "lr": 1e-3, "mu": 0.95, "decay": 0.1, "scale": 0.2 * math.sqrt(max(m, n))}


# ---- the plain forms -----------------------------------------------------------------------------

def _logits(s):
    z = s["X"].float() @ s["W"].float().t()
    return z if s["bias"] is None else z.add_(s["bias"])


def _plain_xent_forward(s):
    # softplus(log sum over the other classes - z_t): lse - z_t itself cancels where a row is sure of its answer
    z = _logits(s)
    t = s["target"].long()
    counts = (t >= 0) & (t < z.shape[1])
    at = torch.where(counts, t, 0)[:, None]
    picked = z.gather(1, at)[:, 0]
    z.scatter_(1, at, torch.where(counts, -math.inf, picked)[:, None])
    top = z.amax(1)
    others = (z - top[:, None]).exp_().sum(1).log_() + top
    d = others - picked
    loss = d.clamp(min=0) + torch.log1p(torch.exp(-d.abs()))
    return {"loss": torch.where(counts, loss, 0.0), "lse": torch.where(counts, torch.logaddexp(others, picked), others)}


def _plain_xent_backward(s):
    t = s["target"].long()
    g = _logits(s).sub_(s["lse"][:, None]).exp_()
    counts = (t >= 0) & (t < g.shape[1])
    g.scatter_add_(1, torch.where(counts, t, 0)[:, None], -counts.float()[:, None])
    g.mul_(torch.where(counts, s["dloss"], 0.0)[:, None])
    dt = s["X"].dtype
    out = {"dX": (g @ s["W"].float()).to(dt), "dW": (g.t() @ s["X"].float()).to(dt)}
    if s["bias"] is not None:
        out["db"] = g.sum(0)
    return out


def _plain_orthogonal(G):
    a, b, c = COEF
    flip = G.shape[1] > G.shape[2]
    X = (G.transpose(1, 2) if flip else G).float()
    norm = X.double().square().sum((1, 2), keepdim=True).sqrt()
    X = torch.where(norm > 0, X.double() / norm, 0.0).float()
    for _ in range(MUON_STEPS):
        A = X @ X.transpose(1, 2).contiguous()
        X = a * X + (b * A + c * (A @ A)) @ X
    return X.transpose(1, 2) if flip else X


def _plain_ortho_update(s):
    g = s["G"].sum(0)
    m = s["momentum"].mul_(s["mu"]).add_(g)
    o = _plain_orthogonal(g + s["mu"] * m)
    s["W"].mul_(1.0 - s["lr"] * s["decay"]).sub_(s["lr"] * s["scale"] * o)
    s["W16"].copy_(s["W"])
    s["Wt16"].copy_(s["W"].transpose(1, 2))
    return {k: s[k] for k in ("W", "W16", "Wt16", "momentum")}


# ---- the framework's calls -----------------------------------------------------------------------

_space = {}


def _workspace(nbytes):
    """The one workspace that a program keeps per stream, as large as the largest call so far needs."""
    if "ws" not in _space or _space["ws"].numel() < nbytes:
        _space["ws"] = torch.empty(max(nbytes, 256), dtype=torch.uint8, device="cuda")
    return _space["ws"].data_ptr(), _space["ws"].numel()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _own_run(s):
    from ctypes import byref, c_size_t

    from tbb_test_amd import capi
    lib, case = capi.lib(), s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    op = case["op"]
    if op.startswith("xent"):
        M, V, K = case["rows"], case["vocab"], case["width"]
        code = capi.MI_BF16 if case["dtype"] == "bf16" else capi.MI_F32
        X, W = s["X"], s["W"]
        if "bytes" not in s:
            fwd, bwd = c_size_t(), c_size_t()
            capi.check(lib.mi_xent_workspace(code, M, V, K, byref(fwd), byref(bwd)))
            s["bytes"] = fwd.value if op == "xent_forward" else bwd.value
        ws, nbytes = _workspace(s["bytes"])
        if op == "xent_forward":
            loss, lse = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
            capi.check(lib.mi_xent_forward(code, M, V, K, X.data_ptr(), K, W.data_ptr(), K, _ptr(s["bias"]),
                                           s["target"].data_ptr(), loss.data_ptr(), lse.data_ptr(), ws, nbytes, stream))
            return {"loss": loss, "lse": lse}
        out = {"dX": torch.empty_like(X), "dW": torch.empty_like(W)}
        if s["bias"] is not None:
            out["db"] = torch.empty(V, device="cuda")
        capi.check(lib.mi_xent_backward(code, M, V, K, X.data_ptr(), K, W.data_ptr(), K, _ptr(s.get("Wt")), V,
                                        _ptr(s["bias"]), s["target"].data_ptr(), s["lse"].data_ptr(),
                                        s["dloss"].data_ptr(), out["dX"].data_ptr(), K, code, out["dW"].data_ptr(), K,
                                        _ptr(out.get("db")), ws, nbytes, stream))
        return out
    b, m, n = case["batch"], case["rows"], case["cols"]
    if "bytes" not in s:
        size = c_size_t()
        capi.check(lib.mi_ortho_workspace(b, m, n, byref(size)))
        s["bytes"] = size.value
    ws, nbytes = _workspace(s["bytes"])
    if op == "orthogonalize":
        code = capi.MI_BF16 if case["dtype"] == "bf16" else capi.MI_F32
        out = torch.empty(b, m, n, dtype=torch.bfloat16, device="cuda")
        capi.check(lib.mi_orthogonalize(code, b, m, n, s["G"].data_ptr(), n, m * n, out.data_ptr(), n, m * n,
                                        MUON_STEPS, ws, nbytes, stream))
        return out
    capi.check(lib.mi_ortho_update_raw(b, m, n, s["W"].data_ptr(), s["W16"].data_ptr(), s["Wt16"].data_ptr(),
                                       s["momentum"].data_ptr(), s["G"].data_ptr(), m * n, b * m * n, case["replicas"],
                                       s["lr"], s["scale"], s["decay"], s["mu"], 1, MUON_STEPS, ws, nbytes, stream))
    return {k: s[k] for k in ("W", "W16", "Wt16", "momentum")}


def run(state):
    if own:
        return _own_run(state)
    op = state["case"]["op"]
    if op == "xent_forward":
        return _plain_xent_forward(state)
    if op == "xent_backward":
        return _plain_xent_backward(state)
    if op == "orthogonalize":
        return _plain_orthogonal(state["G"]).to(torch.bfloat16).contiguous()
    return _plain_ortho_update(state)


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    if case["op"].startswith("xent"):
        M, V, K = case["rows"], case["vocab"], case["width"]
        e = 2 if case["dtype"] == "bf16" else 4
        once = 2.0 * M * V * K
        read = e * (M * K + V * K) + 4 * M + (4 * V if case["bias"] else 0)
        if case["op"] == "xent_forward":
            return {"bytes": read + 8 * M, "flops": once}
        return {"bytes": read + 8 * M + e * (M * K + V * K) + (4 * V if case["bias"] else 0), "flops": 3 * once}
    b, rows, cols = case["batch"], case["rows"], case["cols"]
    m, n = min(rows, cols), max(rows, cols)
    # X X^T and A A are symmetric: one triangle each, then B X
    flops = b * MUON_STEPS * (1.0 * m * m * n + 1.0 * m * m * m + 2.0 * m * m * n)
    if case["op"] == "orthogonalize":
        return {"bytes": b * rows * cols * ((2 if case["dtype"] == "bf16" else 4) + 2), "flops": flops}
    # the gradients once, momentum and W read and written, the two bf16 copies written
    return {"bytes": b * rows * cols * (4 * case["replicas"] + 8 + 8 + 4), "flops": flops}


# ---- the definition in 64 bits -------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"].startswith("xent"):
        M, V = case["rows"], case["vocab"]
        X, W = s["X"].to(f64), s["W"].to(f64)
        bias = torch.zeros(V, dtype=f64, device="cuda") if s["bias"] is None else s["bias"].to(f64)
        step = max(1, (1 << 29) // V)  # rows at a time
        loss, lse, dX = [], [], []
        dW = torch.zeros_like(W) if case["op"] == "xent_backward" else None
        db = torch.zeros_like(bias)
        for i in range(0, M, step):
            x, t = X[i:i + step], s["target"][i:i + step].long()
            z = torch.addmm(bias, x, W.t())
            hit = torch.nn.functional.one_hot(t.clamp(min=0), V).to(torch.bool) & (t >= 0)[:, None]
            if dW is None:
                total = torch.logsumexp(z, 1)
                lse.append(total)
                loss.append(torch.where(t >= 0, total - torch.where(hit, z, 0.0).sum(1), 0.0))
                continue
            d = torch.where(t >= 0, s["dloss"][i:i + step], 0.0).to(f64)
            g = torch.exp(z - s["lse"][i:i + step].to(f64)[:, None])
            g = (g - hit.to(f64)) * d[:, None]
            dX.append(g @ W)
            dW += g.t() @ x
            db += g.sum(0)
        if dW is None:
            return {"loss": torch.cat(loss), "lse": torch.cat(lse)}
        out = {"dX": torch.cat(dX), "dW": dW}
        if s["bias"] is not None:
            out["db"] = db
        return out

    def polar(Y):  # one matrix
        Y = Y / max(float(torch.linalg.matrix_norm(Y)), 1e-300)
        left = Y.shape[0] <= Y.shape[1]
        for _ in range(MUON_STEPS):
            S = Y @ Y.t() if left else Y.t() @ Y
            P = torch.eye(S.shape[0], dtype=f64, device="cuda") * COEF[0] + COEF[1] * S + COEF[2] * (S @ S)
            Y = P @ Y if left else Y @ P
        return Y

    if case["op"] == "orthogonalize":
        return torch.stack([polar(g.to(f64)) for g in s["G"]])
    mu, lr = s["mu"], s["lr"]
    g = s["G"].to(f64).sum(0)
    mom = mu * s["momentum"].to(f64) + g
    o = torch.stack([polar(u) for u in g + mu * mom])
    W = s["W"].to(f64) * (1.0 - lr * s["decay"]) - lr * s["scale"] * o
    return {"W": W, "W16": W, "Wt16": W.transpose(1, 2).contiguous(), "momentum": mom}
