"""Workloads of the dense operators (``similaripy_amd.dense``): embedding rows, score adjustment, distillation from top-k lists.

``own`` false: the operators written out in elementary torch operations, 32 bits whatever the inputs' type, rounded once at the
end.  ``own`` true: the framework's calls.  Sizes are those of this repository's workloads (a catalogue of 100 000 items, the
84 432 items and ~144 ratings per user of MovieLens-32M, 64 entries per row, lists of k = 100 / 200) or generic.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


def listed():
    return [
        # scoring eight requests: one token each, the table's row scaled by sqrt(dim)
        {"name": "embed_single_tokens", "op": "embed", "dtype": "bf16", "n": 8, "vocab": 100_000, "dim": 512, "bag": 0, "ids": "i64"},
        # a training batch of a sequence model: 16 k positions, odd vocabulary
        {"name": "embed_lookup_batch", "op": "embed", "dtype": "bf16", "n": 16_384, "vocab": 84_433, "dim": 1024, "bag": 0, "ids": "i64"},
        # user vectors of a whole slice of users: weighted bags of ~64 items (CSR rows of the rating matrix)
        {"name": "embed_user_bags", "op": "embed", "dtype": "fp32", "n": 65_536, "vocab": 100_000, "dim": 128, "bag": 64, "ids": "i32"},
        # the gradient of the lookup batch: popular tokens repeat hundreds of times
        {"name": "embed_grad_lookup", "op": "embed_grad", "dtype": "bf16", "n": 16_384, "vocab": 84_433, "dim": 1024, "bag": 0, "ids": "i64"},
        # the gradient of weighted bags of MovieLens-like users (mean 144 ratings, some users without any)
        {"name": "embed_grad_bags", "op": "embed_grad", "dtype": "fp32", "n": 8_192, "vocab": 84_432, "dim": 129, "bag": 144, "ids": "i32"},
        # one request: the whole catalogue, its history penalised, a grammar mask of packed bits
        {"name": "adjust_single", "op": "adjust", "dtype": "fp32", "n": 1, "vocab": 100_000, "hist": 300, "penalty": True, "bias": True, "bits": True,
         "filter": 0, "target": 0, "pad": 0, "ids": "i32"},
        # a serving batch: seen items dropped, popularity bias, penalties of each request
        {"name": "adjust_batch", "op": "adjust", "dtype": "bf16", "n": 512, "vocab": 100_000, "hist": 144, "penalty": True, "bias": True, "bits": False,
         "filter": 144, "target": 0, "pad": 0, "ids": "i32"},
        # offline scoring against candidate lists: odd catalogue in padded rows, only listed columns stay
        {"name": "adjust_candidates", "op": "adjust", "dtype": "fp16", "n": 1021, "vocab": 84_431, "hist": 0, "penalty": False, "bias": False, "bits": True,
         "filter": 64, "target": 1000, "pad": 17, "ids": "i32"},
        # a small validation batch against a teacher's 20 best
        {"name": "distill_loss_small", "op": "distill_loss", "dtype": "fp32", "n": 16, "vocab": 10_007, "k": 20, "tau": 2.0, "lse": False, "pad": 0},
        # forward only over a large batch, lists of 100
        {"name": "distill_loss_batch", "op": "distill_loss", "dtype": "bf16", "n": 2048, "vocab": 100_000, "k": 100, "tau": 1.0, "lse": True, "pad": 0},
        # a training step that keeps the rows' statistics between forward and backward, MovieLens catalogue, lists of 200
        {"name": "distill_step", "op": "distill_step", "dtype": "fp32", "n": 1024, "vocab": 84_432, "k": 200, "tau": 2.0, "lse": False, "pad": 0},
        # the same step in one call: loss and gradient from one reading of the scores
        {"name": "distill_loss_grad", "op": "distill_loss_grad", "dtype": "bf16", "n": 4096, "vocab": 100_000, "k": 100, "tau": 1.0, "lse": False, "pad": 0},
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "embed", "embed_grad", "embed_grad", "adjust", "adjust", "adjust", "distill_loss", "distill_step", "distill_loss_grad"])
    dtype = rng.choice(["bf16", "fp32", "fp16"])
    ids = rng.choice(["i32", "i64"])
    if op in ("embed", "embed_grad"):
        bag = rng.choice([0, 0, _log_between(rng, 2, 160)])
        dim = _log_between(rng, 16, 1024)
        if rng.random() < 0.6:
            dim = max(16, dim // 16 * 16)
        vocab = _log_between(rng, 500, 100_000)
        n = _log_between(rng, 1, 16_384 if bag == 0 else max(8, min(65_536, 4_000_000 * 128 // (bag * max(dim, 64)))))
        return {"op": op, "dtype": dtype, "n": n, "vocab": vocab, "dim": dim, "bag": bag, "ids": ids}
    vocab = _log_between(rng, 1000, 100_000)
    pad = rng.choice([0, 0, 1, 8, (-vocab) % 64])
    if op == "adjust":
        n = _log_between(rng, 1, max(2, min(1024, 45_000_000 // vocab)))
        return {"op": op, "dtype": dtype, "n": n, "vocab": vocab, "hist": rng.choice([0, _log_between(rng, 10, 4000)]), "penalty": rng.random() < 0.6,
                "bias": rng.random() < 0.5, "bits": rng.random() < 0.5, "filter": rng.choice([0, _log_between(rng, 8, 1000)]),
                "target": rng.choice([0, 0, _log_between(rng, 8, 1000)]), "pad": pad, "ids": ids}
    n = _log_between(rng, 1, max(2, min(4096, 80_000_000 // vocab)))
    return {"op": op, "dtype": dtype, "n": n, "vocab": vocab, "k": _log_between(rng, 5, 256), "tau": rng.choice([1.0, 2.0, 4.0]), "lse": rng.random() < 0.3, "pad": pad}


# ---- inputs ------------------------------------------------------------------------------------------------------------------

def _popularity(vocab):
    p = 1.0 / np.arange(1, vocab + 1) ** 0.9            # Zipf(0.9), as the repository's MovieLens-like matrix
    return np.cumsum(p / p.sum())


def _popular_ids(gen, vocab, count):
    """`count` ids of a shuffled catalogue with Zipf popularity."""
    cdf = torch.from_numpy(_popularity(vocab)).cuda()
    rank = torch.searchsorted(cdf, torch.rand(count, generator=gen, device="cuda", dtype=torch.float64)).clamp_(max=vocab - 1)
    return torch.randperm(vocab, generator=gen, device="cuda")[rank]


def _ragged(gen, n, mean, empty):
    """Row pointers of n rows with log-normal lengths (user activity), about `empty` of them empty."""
    act = torch.exp(torch.randn(n, generator=gen, device="cuda"))
    lens = (act * (mean / math.exp(0.5))).round().clamp_(1, 16 * mean).long()
    lens[torch.rand(n, generator=gen, device="cuda") < empty] = 0
    indptr = torch.zeros(n + 1, dtype=torch.int64, device="cuda")
    indptr[1:] = torch.cumsum(lens, 0)
    return indptr


def _lists(gen, n_rows, vocab, mean, it):
    """A CSR pattern: row pointers and ids (popular ids repeat inside a row, as tokens of a history do)."""
    indptr = _ragged(gen, n_rows, mean, 0.05)
    total = int(indptr[-1])
    return {"indptr": indptr.to(it), "indices": _popular_ids(gen, vocab, total).to(it), "total": total}


def _of_targets(csr, targets):
    """Where the entries of the listed rows lie, for the plain form: (row of each entry, id of each entry)."""
    lens = (csr["indptr"][1:] - csr["indptr"][:-1])[targets]
    csr["taken"] = int(lens.sum())


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    op, n, vocab = case["op"], case["n"], case["vocab"]
    if op in ("embed", "embed_grad"):
        it = torch.int32 if case["ids"] == "i32" else torch.int64
        dim, s = case["dim"], {"op": op, "vocab": vocab, "n": n, "scale": math.sqrt(case["dim"]) if case["bag"] == 0 else 1.0}
        if case["bag"]:
            indptr = _ragged(gen, n, case["bag"], 0.02)
            total = int(indptr[-1])
            s["indptr"], s["weights"] = indptr.to(it), torch.rand(total, generator=gen, device="cuda") * 0.2
        else:
            total, s["indptr"], s["weights"] = n, None, None
        s["indices"] = _popular_ids(gen, vocab, total).to(it)
        if op == "embed":
            s["table"] = (torch.randn(vocab, dim, generator=gen, device="cuda") / math.sqrt(dim)).to(dt)
        else:
            s["grad"] = (torch.randn(n, dim, generator=gen, device="cuda") * 0.02).to(dt)
        return s
    stored = torch.empty(n, vocab + case["pad"], device="cuda", dtype=dt)
    for a in range(0, n, 256):
        stored[a:a + 256] = torch.randn(min(256, n - a), vocab + case["pad"], generator=gen, device="cuda") * 2.5
    if op == "adjust":
        it = torch.int32 if case["ids"] == "i32" else torch.int64
        rows = 4 * n                                     # the CSR rows of all users; the batch names its own
        s = {"op": op, "scores": stored[:, :vocab], "targets": torch.randperm(rows, generator=gen, device="cuda")[:n].to(it),
             "repetition": None, "presence": None, "frequency": None, "history": None, "filter": None, "target": None, "bias": None, "bits": None}
        if case["hist"]:
            s["history"] = _lists(gen, rows, vocab, case["hist"], it)
        if case["penalty"]:
            s["repetition"] = 1.0 + 0.5 * torch.rand(n, generator=gen, device="cuda")
            s["presence"] = 0.3 * torch.rand(n, generator=gen, device="cuda")
            s["frequency"] = 0.1 * torch.rand(n, generator=gen, device="cuda")
        if case["filter"]:
            s["filter"] = _lists(gen, rows, vocab, case["filter"], it)
        if case["target"]:
            s["target"] = _lists(gen, rows, vocab, case["target"], it)
        for name in ("history", "filter", "target"):
            if s[name] is not None:
                _of_targets(s[name], s["targets"].long())
        if case["bias"]:
            s["bias"] = -0.3 * torch.rand(vocab, generator=gen, device="cuda")
        if case["bits"]:
            words = (vocab + 31) // 32
            s["bits"] = torch.randint(-2**31, 2**31, (n, words), generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
        return s
    k = case["k"]
    at = (torch.arange(k, device="cuda") + torch.rand(n, k, generator=gen, device="cuda")) * (vocab / k)
    cols = at.long().clamp_(max=vocab - 1)
    cols = cols.gather(1, torch.rand(n, k, generator=gen, device="cuda").argsort(1))
    values = (torch.randn(n, k, generator=gen, device="cuda") * 2.0 + 6.0).sort(1, descending=True).values
    counts = torch.full((n,), k, device="cuda", dtype=torch.int32)
    short = torch.rand(n, generator=gen, device="cuda") < 0.1
    counts[short] = torch.randint(0, k + 1, (n,), generator=gen, device="cuda", dtype=torch.int32)[short]
    near = stored.gather(1, cols) + (0.5 * values).to(dt)                     # the student has learnt some of it
    stored.scatter_(1, cols, near)
    lse = torch.logsumexp(values / case["tau"], 1) + 0.5 * torch.rand(n, generator=gen, device="cuda") if case["lse"] else None
    return {"op": op, "student": stored[:, :vocab], "cols": cols.to(torch.int32), "values": values, "counts": counts, "tau": case["tau"], "lse": lse,
            "grad_loss": torch.full((n,), 1.0 / n, device="cuda")}


# ---- one pass ----------------------------------------------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from similaripy_amd import dense
    if s["op"] == "embed":
        return dense.embed_rows(s["table"], s["indices"], s["indptr"], s["weights"], scale=s["scale"])
    if s["op"] == "embed_grad":
        return dense.embed_rows_grad(s["grad"], s["indices"], s["vocab"], s["indptr"], s["weights"], scale=s["scale"])
    if s["op"] == "adjust":
        pair = lambda c: None if c is None else (c["indptr"], c["indices"])  # noqa: E731
        kw = {} if s["repetition"] is None else {"repetition": s["repetition"], "presence": s["presence"], "frequency": s["frequency"]}
        return dense.adjust_scores(s["scores"], targets=s["targets"], history=pair(s["history"]), bias=s["bias"], allowed=s["bits"],
                                   filter_cols=pair(s["filter"]), target_cols=pair(s["target"]), **kw)
    lists = (s["cols"], s["values"], s["counts"])
    if s["op"] == "distill_loss":
        return dense.distill_loss(s["student"], *lists, temperature=s["tau"], teacher_lse=s["lse"])
    if s["op"] == "distill_step":
        loss, stats = dense.distill_loss(s["student"], *lists, temperature=s["tau"], teacher_lse=s["lse"], return_stats=True)
        return loss, dense.distill_grad(s["student"], stats, *lists, grad_loss=s["grad_loss"], temperature=s["tau"], teacher_lse=s["lse"])
    return dense.distill_loss_grad(s["student"], *lists, grad_loss=s["grad_loss"], temperature=s["tau"], teacher_lse=s["lse"])


def _entry_rows(s):
    """The output row of every entry of a CSR."""
    lens = s["indptr"][1:] - s["indptr"][:-1]
    return torch.repeat_interleave(torch.arange(s["n"], device="cuda"), lens.long(), output_size=s["indices"].numel())


def _counted(csr, targets, scores):
    """How often row targets[b] of the CSR lists column v: [b, v]."""
    lens = (csr["indptr"][1:] - csr["indptr"][:-1])[targets].long()
    ends = torch.cumsum(lens, 0)
    row = torch.repeat_interleave(torch.arange(lens.numel(), device="cuda"), lens, output_size=csr["taken"])
    at = torch.arange(csr["taken"], device="cuda") - (ends - lens)[row] + csr["indptr"][targets].long()[row]
    found = torch.zeros(scores.shape, dtype=torch.int32, device="cuda")
    found.index_put_((row, csr["indices"][at].long()), torch.ones((), dtype=torch.int32, device="cuda"), accumulate=True)
    return found


def _run_plain(s):
    if s["op"] == "embed":
        if s["indptr"] is None:
            return (s["table"][s["indices"]].float() * s["scale"]).to(s["table"].dtype)
        out = torch.zeros(s["n"], s["table"].shape[1], device="cuda")
        out.index_add_(0, _entry_rows(s), s["table"][s["indices"]].float() * s["weights"][:, None])
        return (out * s["scale"]).to(s["table"].dtype)
    if s["op"] == "embed_grad":
        out = torch.zeros(s["vocab"], s["grad"].shape[1], device="cuda")
        each = s["grad"].float() if s["indptr"] is None else s["grad"][_entry_rows(s)].float() * s["weights"][:, None]
        out.index_add_(0, s["indices"], each)
        return (out * s["scale"]).to(s["grad"].dtype)
    if s["op"] == "adjust":
        scores, targets = s["scores"], s["targets"].long()
        y = scores.float()
        if s["history"] is not None and s["repetition"] is not None:
            c = _counted(s["history"], targets, scores)
            r = s["repetition"][:, None]
            fined = torch.where(y > 0, y / r, y * r) - (s["presence"][:, None] + s["frequency"][:, None] * c)
            y = torch.where(c > 0, fined, y)
        if s["bias"] is not None:
            y = y + s["bias"]
        gone = torch.zeros(y.shape, dtype=torch.bool, device="cuda")
        if s["filter"] is not None:
            gone |= _counted(s["filter"], targets, scores) > 0
        if s["target"] is not None:
            gone |= _counted(s["target"], targets, scores) == 0
        if s["bits"] is not None:
            col = torch.arange(y.shape[1], device="cuda")
            gone |= ((s["bits"][:, col // 32] >> (col % 32)) & 1) == 0
        return y.masked_fill(gone, -math.inf).to(scores.dtype)
    z, tau, cols = s["student"].float() / s["tau"], s["tau"], s["cols"].long()
    listed_ = torch.arange(cols.shape[1], device="cuda") < s["counts"][:, None]
    t = torch.where(listed_, s["values"] / tau, -math.inf)
    if s["lse"] is None:
        top = t.max(1, keepdim=True).values.clamp(min=-3e38)
        weight = torch.exp(t - top)
        total = weight.sum(1, keepdim=True)
        p = weight / total.clamp(min=1e-30)
        logp = t - top - torch.log(total.clamp(min=1e-30))
    else:
        logp = t - s["lse"][:, None]
        p = torch.exp(logp)
    high = z.max(1, keepdim=True).values
    e = torch.exp(z - high)
    z_sum = e.sum(1, keepdim=True)
    logq = z.gather(1, cols) - high - torch.log(z_sum)
    loss = tau * tau * torch.where(p > 0, p * (logp - logq), 0.0).sum(1)
    if s["op"] == "distill_loss":
        return loss
    grad = e * (p.sum(1, keepdim=True) / z_sum)
    grad.scatter_add_(1, cols, -p)
    return loss, (grad * (s["grad_loss"] * tau)[:, None]).to(s["student"].dtype)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------

def work(case):
    op, n, vocab, b = case["op"], case["n"], case["vocab"], BYTES[case["dtype"]]
    if op in ("embed", "embed_grad"):
        idb = 4 if case["ids"] == "i32" else 8
        entries = n * (case["bag"] or 1)
        p = np.diff(_popularity(vocab), prepend=0.0)
        touched = float((-np.expm1(entries * np.log1p(-p))).sum())             # distinct ids expected among the entries
        side = entries * (idb + (4 if case["bag"] else 0)) + (n * idb if case["bag"] else 0)
        rows = touched + n if op == "embed" else n + vocab
        return {"bytes": side + rows * case["dim"] * b, "flops": 2.0 * entries * case["dim"]}
    if op == "adjust":
        idb = 4 if case["ids"] == "i32" else 8
        hist = case["hist"] if case["penalty"] else 0
        lists = n * idb * (hist + case["filter"] + case["target"])
        side = lists + (4 * vocab if case["bias"] else 0) + (n * vocab / 8 if case["bits"] else 0)
        return {"bytes": 2.0 * n * vocab * b + side, "flops": 4.0 * n * vocab}
    passes = 1 if op == "distill_loss" else 2
    return {"bytes": passes * n * vocab * b + n * (8.0 * case["k"] + 12), "flops": (4.0 if passes == 1 else 7.0) * n * vocab}


# ---- the same from the definitions, in 64 bits -------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op, n, vocab = case["op"], case["n"], case["vocab"]
    if op in ("embed", "embed_grad"):
        ids = s["indices"].long()
        if op == "embed" and s["indptr"] is None:
            return torch.index_select(s["table"].double(), 0, ids).mul_(s["scale"])
        if s["indptr"] is None:
            row, w, bounds = torch.arange(n, device="cuda"), torch.ones(n, device="cuda", dtype=torch.float64), None
        else:
            bounds = s["indptr"].long()
            row = torch.bucketize(torch.arange(ids.numel(), device="cuda"), bounds[1:], right=True)
            w = s["weights"].double()
        if op == "embed":
            source, order = s["table"], torch.arange(ids.numel(), device="cuda")
            pick = ids
        else:
            source, order = s["grad"], torch.argsort(ids, stable=True)
            pick, w = row[order], w[order]
            bounds = torch.searchsorted(ids[order], torch.arange(vocab + 1, device="cuda"))
        out = torch.empty(bounds.numel() - 1, case["dim"], device="cuda", dtype=torch.float64)
        for c in range(0, case["dim"], 16):              # sums of segments as differences of running sums
            part = torch.zeros(pick.numel() + 1, min(16, case["dim"] - c), device="cuda", dtype=torch.float64)
            torch.cumsum(source[:, c:c + 16].double()[pick] * w[:, None], 0, out=part[1:])
            out[:, c:c + 16] = part[bounds[1:]] - part[bounds[:-1]]
        return out * s["scale"]
    if op == "adjust":
        out = torch.empty(n, vocab, device="cuda", dtype=torch.float64)
        tell = s["targets"].tolist()
        ptr = {name: s[name]["indptr"].tolist() for name in ("history", "filter", "target") if s[name] is not None}

        def count(name, i):
            a, e = ptr[name][tell[i]], ptr[name][tell[i] + 1]
            return torch.bincount(s[name]["indices"][a:e].long(), minlength=vocab)

        for i in range(n):
            y = s["scores"][i].double()
            if s["history"] is not None and s["repetition"] is not None:
                c = count("history", i).double()
                r, hit = s["repetition"][i].double(), c > 0
                y = torch.where(hit & (y > 0), y / r, torch.where(hit, y * r, y))
                y = y - hit * s["presence"][i].double() - c * s["frequency"][i].double()
            if s["bias"] is not None:
                y = y + s["bias"].double()
            if s["filter"] is not None:
                y[count("filter", i) > 0] = -math.inf
            if s["target"] is not None:
                y[count("target", i) == 0] = -math.inf
            if s["bits"] is not None:
                word = s["bits"][i].long() & 0xFFFFFFFF
                bit = (word[:, None] // (2 ** torch.arange(32, device="cuda"))[None, :]) % 2
                y[bit.reshape(-1)[:vocab] == 0] = -math.inf
            out[i] = y
        return out
    tau, loss = float(case["tau"]), torch.empty(n, device="cuda", dtype=torch.float64)
    grad = None if op == "distill_loss" else torch.empty(n, vocab, device="cuda", dtype=torch.float64)
    for a in range(0, n, 128):
        part = slice(a, min(n, a + 128))
        logq = torch.log_softmax(s["student"][part].double() / tau, 1)
        cols, count = s["cols"][part].long(), s["counts"][part].long()
        ok = torch.arange(cols.shape[1], device="cuda")[None, :].expand_as(cols) < count[:, None]
        t = (s["values"][part].double() / tau).masked_fill(~ok, -math.inf)
        logp = torch.log_softmax(t, 1) if s["lse"] is None else t - s["lse"][part].double()[:, None]
        p = torch.where(ok, logp.exp(), 0.0)
        mine = torch.where(ok, logq.gather(1, cols), 0.0)
        loss[part] = tau * tau * (p * (torch.where(ok, logp, 0.0) - mine)).sum(1)
        if grad is not None:
            full = torch.zeros_like(logq).scatter_add_(1, cols, p)
            grad[part] = (logq.exp() * p.sum(1, keepdim=True) - full) * tau * s["grad_loss"][part].double()[:, None]
    return loss if grad is None else (loss, grad)
