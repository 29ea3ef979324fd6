"""Layer norm, dropout and the classifier with its softmax cost: cases, inputs, plain forms and values in 64 bits.

All matrices are (features, cases) with the cases contiguous, in float32, as everywhere in this framework.  Three operators:

  norm     y = gain (x - mean) r + bias over the features of each case, and its gradients
  dropout  target = scaleTargets target + x keep / (1 - p), keep from a counter-based generator (the gradient is the same call)
  cost     a fully connected layer under a softmax and a logreg cost, without the (classes, cases) matrix; "train" adds the
           gradients of the inputs, weights and biases
"""
import math

import numpy as np
import torch

own = False
EPS = 1e-5


def listed():
    return [
        # one image's 512-value feature vector (DeepID2+ fc5) normalised when it is served
        {"name": "norm_one_case", "op": "norm", "features": 512, "cases": 1, "undo": False},
        # whole 55x55x3 images normalised ahead of a net, one minibatch
        {"name": "norm_images", "op": "norm", "features": 9075, "cases": 128, "undo": False},
        # the training step's normalisation of a 512-value feature layer, one minibatch
        {"name": "norm_undo_minibatch", "op": "norm", "features": 512, "cases": 128, "undo": True},
        # an odd number of classes normalised over a ragged last minibatch
        {"name": "norm_undo_odd", "op": "norm", "features": 4213, "cases": 509, "undo": True},
        # a wide layer over a large batch: bound by memory
        {"name": "norm_undo_large", "op": "norm", "features": 4096, "cases": 16384, "undo": True},
        # dropout behind the 160-value feature layer, one minibatch: latency
        {"name": "dropout_minibatch", "op": "dropout", "features": 160, "cases": 128, "p": 0.4, "add": False},
        # the gradient added onto one that is there, an odd number of elements
        {"name": "dropout_add_odd", "op": "dropout", "features": 4213, "cases": 509, "p": 0.1, "add": True},
        # the maps of a conv layer over a large batch: bound by memory
        {"name": "dropout_large", "op": "dropout", "features": 8192, "cases": 16384, "p": 0.4, "add": False},
        # the cost of one image over the identities of DeepID
        {"name": "cost_one_case", "op": "cost", "inputs": 160, "outputs": 4213, "cases": 1, "train": False, "padded": 0, "masked": False},
        # the cost of a ragged, padded batch over the identities of DeepID2+
        {"name": "cost_ragged", "op": "cost", "inputs": 512, "outputs": 10575, "cases": 509, "train": False, "padded": 13, "masked": True},
        # one training minibatch of DeepID2+
        {"name": "train_minibatch", "op": "cost", "inputs": 512, "outputs": 10575, "cases": 128, "train": True, "padded": 0, "masked": False},
        # one large training batch over many identities
        {"name": "train_large", "op": "cost", "inputs": 512, "outputs": 100000, "cases": 1024, "train": True, "padded": 0, "masked": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "dropout", "cost", "cost", "cost"])
    if op == "norm":
        features = _log_int(rng, 2, 20000)
        return {"op": op, "features": features, "cases": _log_int(rng, 1, min(20000, (1 << 26) // features)), "undo": rng.random() < 0.6}
    if op == "dropout":
        features = _log_int(rng, 1, 20000)
        return {"op": op, "features": features, "cases": _log_int(rng, 1, min(20000, (1 << 26) // features)),
                "p": rng.choice([0.0, 0.1, 0.25, 0.4, 0.5, 0.9]), "add": rng.random() < 0.5}
    inputs, outputs = _log_int(rng, 16, 2048), _log_int(rng, 2, 100000)
    cases = _log_int(rng, 1, min(2048, 100000 * 512 * 1024 // (inputs * outputs)))
    return {"op": op, "inputs": inputs, "outputs": outputs, "cases": cases, "train": rng.random() < 0.6,
            "padded": rng.choice([0, 0, cases // 5]), "masked": outputs > 8 and rng.random() < 0.3}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = dict(case)
    if case["op"] == "norm":
        f, n = case["features"], case["cases"]
        # activations of a layer: every case with an offset and a scale of its own
        s["x"] = normal(f, n) * (0.5 + torch.rand(n, generator=g, device="cuda") * 2) + normal(n) * 2
        s["gain"], s["bias"] = 1 + 0.2 * normal(f), 0.2 * normal(f)
        if case["undo"]:
            s["g"] = normal(f, n) / n
    elif case["op"] == "dropout":
        f, n = case["features"], case["cases"]
        s["x"] = normal(f, n)
        s["seed"], s["step"] = (seed * 0x9E3779B97F4A7C15 + 12345) % (1 << 63), 1000 + seed % 7919
        if case["add"]:
            s["there"] = normal(f, n)
    else:
        d, v, n = case["inputs"], case["outputs"], case["cases"]
        s["w"] = normal(v, d) / math.sqrt(d)
        s["b"] = 0.1 * normal(v)
        labels = torch.randint(v, (n,), generator=g, device="cuda")
        # features that lean towards their class, as those of a net in the middle of its training
        s["x"] = normal(d, n) + (8 / (1 + 4 / math.sqrt(d))) * s["w"][labels].t()
        if case["masked"]:  # classes that take no part in this batch
            hidden = torch.rand(v, generator=g, device="cuda") < 0.02
            hidden[labels] = False
            s["b"] = torch.where(hidden, torch.full_like(s["b"], -math.inf), s["b"])
        if case["padded"]:  # cases behind the last image: no label
            labels[n - case["padded"]:] = -1
        s["labels"] = labels.float()
        s["coeff"] = 1.0 / n
    if own:
        _buffers(s)
    return s


# ---------------------------------------------------------------------------------------------- the framework's calls
def _lib():
    import ccn_loader
    ccn_loader.load()
    from cuda_convnet_amd import capi
    return capi.lib()


def _buffers(s):
    """What a program allocates once: output matrices and the workspace."""
    lib = s["lib"] = _lib()

    def empty(*shape):
        return torch.empty(*shape, device="cuda")

    if s["op"] == "norm":
        f, n = s["features"], s["cases"]
        size = lib.raw("mcn_layer_norm_workspace_bytes")(f, n)
        s["y"], s["stats"] = empty(f, n), empty(2, n)
        if s["undo"]:
            size = max(size, lib.raw("mcn_layer_norm_undo_workspace_bytes")(f, n))
            s["dx"], s["dgain"], s["dbias"] = empty(f, n), empty(f), empty(f)
    elif s["op"] == "dropout":
        size = 0
        s["y"] = empty(s["features"], s["cases"])
    else:
        d, v, n = s["inputs"], s["outputs"], s["cases"]
        size = lib.raw("mcn_fc_logreg_workspace_bytes")(d, v, n, 1 if s["train"] else 0)
        s["stats"], s["logp"], s["correct"] = empty(2, n), empty(n), empty(n)
        if s["train"]:
            s["dx"], s["dw"], s["db"] = empty(d, n), empty(v, d), empty(v)
    s["ws"], s["size"] = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda"), size


def _run_own(s):
    lib, stream = s["lib"], torch.cuda.current_stream().cuda_stream
    p = {k: t.data_ptr() for k, t in s.items() if isinstance(t, torch.Tensor)}
    if s["op"] == "norm":
        f, n = s["features"], s["cases"]
        lib.call("mcn_layer_norm", p["x"], p["gain"], p["bias"], p["y"], p["stats"], f, n, EPS, p["ws"], s["size"], stream)
        if not s["undo"]:
            return {"y": s["y"], "stats": s["stats"]}
        lib.call("mcn_layer_norm_undo", p["g"], p["x"], p["gain"], p["stats"], p["dx"], p["dgain"], p["dbias"], f, n,
                 0.0, 1.0, 0.0, 1.0, 0.0, 1.0, p["ws"], s["size"], stream)
        return {"y": s["y"], "stats": s["stats"], "dx": s["dx"], "dgain": s["dgain"], "dbias": s["dbias"]}
    if s["op"] == "dropout":
        if s["add"]:
            s["y"].copy_(s["there"])
        lib.call("mcn_dropout", p["x"], p["y"], s["x"].numel(), s["p"], s["seed"], s["step"], None, 1.0 if s["add"] else 0.0, 1.0, stream)
        return s["y"]
    d, v, n = s["inputs"], s["outputs"], s["cases"]
    lib.call("mcn_fc_logreg_cost", p["w"], p["x"], p["b"], p["labels"], p["stats"], p["logp"], p["correct"], d, v, n, None,
             p["ws"], s["size"], stream)
    out = {"stats": s["stats"], "logp": s["logp"], "correct": s["correct"]}
    if s["train"]:
        lib.call("mcn_fc_logreg_grad", p["w"], p["x"], p["b"], p["labels"], p["stats"], p["dx"], p["dw"], p["db"], d, v, n, s["coeff"],
                 0.0, 0.0, 1.0, 0.0, 1.0, p["ws"], s["size"], stream)
        out.update(dx=s["dx"], dw=s["dw"], db=s["db"])
    return out


# ------------------------------------------------------------------------------------------------------ the plain forms
def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "norm":
        return _norm(s)
    if s["op"] == "dropout":
        keep = _keep(s["x"].numel(), s["p"], s["seed"], s["step"], s["x"].device).view_as(s["x"])
        y = torch.where(keep, s["x"] * _dropout_scale(s["p"]), torch.zeros_like(s["x"]))
        return s["there"] + y if s["add"] else y
    return _cost(s)


def _norm(s):
    x, gain = s["x"], s["gain"][:, None]
    mean = x.mean(0)
    centred = x - mean
    r = 1 / torch.sqrt((centred * centred).mean(0) + EPS)
    hat = centred * r
    out = {"y": gain * hat + s["bias"][:, None], "stats": torch.stack([mean, r])}
    if s["undo"]:
        h = gain * s["g"]
        out["dx"] = r * (h - h.mean(0) - hat * (h * hat).mean(0))
        out["dgain"] = (s["g"] * hat).sum(1)
        out["dbias"] = s["g"].sum(1)
    return out


def _dropout_scale(p):
    return float(np.float32(1 / (1 - float(np.float32(p)))))


def _keep(count, p, seed, step, device):
    """Philox-4x32 with ten rounds (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; SC 2011): the counter is
    (element / 4, step), the key the seed; element e takes word e % 4 and is kept where that is at least floor(p 2^32)."""
    mask = 0xFFFFFFFF
    quad = torch.arange((count + 3) // 4, dtype=torch.int64, device=device)
    c0, c1 = quad & mask, quad >> 32
    c2, c3 = torch.full_like(quad, step & mask), torch.full_like(quad, step >> 32)
    k0, k1 = seed & mask, seed >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & mask) ^ c1 ^ k0, b & mask, ((a >> 32) & mask) ^ c3 ^ k1, a & mask
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    words = torch.stack([c0, c1, c2, c3], 1).view(-1)[:count]
    return words >= math.floor(float(np.float32(p)) * 2.0 ** 32)


def _cost(s):
    z = s["w"] @ s["x"] + s["b"][:, None]
    v, n = z.shape
    counts = (s["labels"] >= 0) & (s["labels"] < v)
    label = torch.where(counts, s["labels"], torch.zeros_like(s["labels"])).long()
    top = z.max(0).values
    e = torch.exp(z - top)
    total = e.sum(0)
    at = z.gather(0, label[None])[0]
    zero = torch.zeros_like(total)
    out = {"stats": torch.stack([top, total]),
           "logp": torch.where(counts, at - top - torch.log(total), zero),
           "correct": torch.where(counts & (at == top), 1 / (z == top).sum(0).float(), zero)}
    if s["train"]:
        grad = -e / total
        grad[label, torch.arange(n, device=z.device)] += 1
        grad = grad * (s["coeff"] * counts.float())
        out.update(dx=s["w"].t() @ grad, dw=grad @ s["x"].t(), db=grad.sum(1))
    return out


# ------------------------------------------------------------------------------------------------------ values in 64 bits
def exact(case, seed):
    s = {k: t.double() if isinstance(t, torch.Tensor) else t for k, t in prepare(case, seed).items() if k not in ("lib", "ws")}
    if case["op"] == "norm":
        f = case["features"]
        mean = s["x"].sum(0) / f
        var = ((s["x"] - mean) ** 2).sum(0) / f
        std = (var + EPS).sqrt()
        y = s["gain"].view(-1, 1) * ((s["x"] - mean) / std) + s["bias"].view(-1, 1)
        out = {"y": y, "stats": torch.stack([mean, 1 / std])}
        if case["undo"]:
            # through the mean and the variance, term by term
            hat, dhat = (s["x"] - mean) / std, s["g"] * s["gain"].view(-1, 1)
            dvar = (dhat * (s["x"] - mean)).sum(0) * -0.5 / std ** 3
            dmean = -dhat.sum(0) / std
            out["dx"] = dhat / std + dvar * 2 * (s["x"] - mean) / f + dmean / f
            out["dgain"], out["dbias"] = (s["g"] * hat).sum(1), s["g"].sum(1)
        return out
    if case["op"] == "dropout":
        p = float(np.float32(case["p"]))
        kept = _kept_words(s["x"].numel(), s["seed"], s["step"]) >= int(p * 4294967296)
        y = s["x"] * torch.from_numpy(kept).to(s["x"].device).view_as(s["x"]) / (1 - p)
        return s["there"] + y if case["add"] else y
    v, n = case["outputs"], case["cases"]
    z = torch.addmm(s["b"].view(-1, 1), s["w"], s["x"])
    used = ((s["labels"] >= 0) & (s["labels"] < v)).double()
    label = s["labels"].clamp(0, v - 1).long()
    lse = torch.logsumexp(z, 0)
    top, _ = torch.max(z, 0)
    at = z[label, torch.arange(n, device=z.device)]
    ties = (z == top).double().sum(0)
    out = {"stats": torch.stack([top, torch.exp(lse - top)]), "logp": (at - lse) * used, "correct": (at == top).double() / ties * used}
    if case["train"]:
        z.sub_(lse).exp_().neg_()  # minus the probabilities, in place: the matrix is large
        z[label, torch.arange(n, device=z.device)] += 1
        z.mul_(used * s["coeff"])
        out.update(dx=torch.mm(s["w"].t(), z), dw=torch.mm(z, s["x"].t()), db=z.sum(1))
    return out


def _kept_words(count, seed, step):
    """The generator's words for `count` elements, by numpy's unsigned arithmetic."""
    quads = (count + 3) // 4
    words = np.empty((quads, 4), np.uint32)
    low = np.uint64(0xFFFFFFFF)
    with np.errstate(over="ignore"):
        for start in range(0, quads, 1 << 15):
            q = np.arange(start, min(quads, start + (1 << 15)), dtype=np.uint64)
            ctr = [q & low, q >> np.uint64(32), np.full_like(q, step & 0xFFFFFFFF), np.full_like(q, step >> 32)]
            key = [np.uint64(seed & 0xFFFFFFFF), np.uint64(seed >> 32)]
            for _ in range(10):
                first, second = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
                ctr = [(second >> np.uint64(32)) ^ ctr[1] ^ key[0], second & low, (first >> np.uint64(32)) ^ ctr[3] ^ key[1], first & low]
                key = [(key[0] + np.uint64(0x9E3779B9)) & low, (key[1] + np.uint64(0xBB67AE85)) & low]
            words[start:start + len(q)] = np.stack(ctr, 1).astype(np.uint32)
    return words.reshape(-1)[:count]


# ------------------------------------------------------------------------------------------------------ what cannot be done without
def work(case):
    if case["op"] == "norm":
        e, f, n = case["features"] * case["cases"], case["features"], case["cases"]
        if case["undo"]:  # forward and backward: x read, y written; x and g read, dx written
            return {"bytes": 4 * (4 * e + 5 * f + 2 * n), "flops": 22 * e}
        return {"bytes": 4 * (2 * e + 2 * f + 2 * n), "flops": 8 * e}
    if case["op"] == "dropout":
        e = case["features"] * case["cases"]
        return {"bytes": 4 * e * (3 if case["add"] else 2), "flops": 3 * e}
    d, v, n = case["inputs"], case["outputs"], case["cases"]
    if case["train"]:
        return {"bytes": 4 * (2 * v * d + 2 * d * n + 2 * v + 5 * n), "flops": 6 * v * d * n + 12 * v * n}
    return {"bytes": 4 * (v * d + d * n + v + 5 * n), "flops": 2 * v * d * n + 6 * v * n}
