"""Performance cases of the operators on a recognizer's logits.

A recognizer ends in one row of class logits per time step.  Three operators
work on such rows, in fp32 or bf16, on the caller's device memory:

* ``rules``: penalties for classes in a row's history, class biases and masks
  of allowed classes, written to a second tensor;
* ``top``: the k best classes of each row (under the rules, where given) and
  the log-sum-exp of all others at a temperature;
* ``distill``: the loss of a student's rows against a teacher's top logits and
  its gradient, in one call ("both") or apart ("loss", "grad").

Classes are the recognizers' (6906 and 18710) and generic larger or odd ones;
rows are time steps: 40 a line of 320 pixels, 63 of 500, batches of 1, 6, 64
and 256 lines, and 256 sequences decoded token by token.

Plain forms are elementary torch operations in 32 bits; ``exact`` restates the
definitions in 64 bits.
"""

import math
import pathlib
import random
import sys

import torch

own = False

INF = float("inf")
_kept = {}


# ------------------------------------------------------------------- cases

def _rules(name, rows, classes, dtype="f32", pad=0, steps=1, masks="none", bias="none", history=0):
    """``masks``: none, one for all rows, or one per line of ``steps`` rows;
    ``bias`` likewise; ``history``: longest history of a row (0: no
    penalties); ``pad``: elements between rows."""
    return {"name": name, "op": "rules", "rows": rows, "classes": classes, "dtype": dtype, "pad": pad,
            "steps": steps, "masks": masks, "bias": bias, "history": history}


def _top(name, rows, classes, k, dtype="f32", pad=0, steps=1, masks="none", tau=1.0):
    return {"name": name, "op": "top", "rows": rows, "classes": classes, "dtype": dtype, "pad": pad,
            "steps": steps, "masks": masks, "bias": "none", "history": 0, "k": k, "tau": tau}


def _distill(name, rows, classes, k, mode, dtype="f32", pad=0, steps=40, tau=1.0, rest=True):
    return {"name": name, "op": "distill", "rows": rows, "classes": classes, "dtype": dtype, "pad": pad,
            "steps": steps, "k": k, "tau": tau, "rest": rest, "mode": mode}


def listed():
    return [
        # One decoded token: penalties for what the line says already.  The
        # smallest call, bound by its launch.
        _rules("rules_step", 1, 6906, history=25),
        # A batch of lines, each with its own grammar, under a lexicon's bias.
        _rules("rules_lines", 64 * 40, 6906, steps=40, masks="line", bias="all"),
        # One engine batch of a page in one script, rows of a padded tensor.
        _rules("rules_page_bf16", 6 * 63, 18710, "bf16", pad=3, steps=63, masks="all", bias="all"),
        # A decoding step of 256 sequences over a large vocabulary.
        _rules("rules_decode_bf16", 256, 131072, "bf16", masks="line", history=2000),
        # Candidates of a single step.
        _top("top_step", 1, 18710, 5),
        # Candidates of a page's lines, each under its grammar.
        _top("top_masked", 6 * 63, 18710, 3, steps=63, masks="line"),
        # A teacher's targets for a batch of lines.
        _top("top_teacher", 64 * 40, 18710, 32, tau=2.0),
        # The same for a bulk batch in bf16, wide lists.
        _top("top_teacher_bf16", 256 * 40, 18710, 64, "bf16"),
        # A training step's loss and gradient on a single line, edge tier.
        _distill("distill_line", 40, 6906, 8, "both"),
        # Validation: the loss alone.
        _distill("distill_loss", 64 * 40, 18710, 32, "loss", tau=2.0),
        # The backward pass behind a loss computed earlier.
        _distill("distill_grad", 64 * 40, 18710, 32, "grad", tau=2.0),
        # A bulk training step in bf16: the largest call.
        _distill("distill_b256_bf16", 256 * 40, 18710, 64, "both", "bf16"),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    while True:
        op = rng.choice(("rules", "top", "distill"))
        dtype = rng.choice(("f32", "bf16"))
        classes = rng.choice((6906, 18710, log_int(97, 131072), log_int(97, 131072)))
        steps = rng.choice((1, 40, 63, log_int(2, 200)))
        rows = steps * log_int(1, max(1, 10240 // steps))
        pad = rng.choice((0, 0, rng.randint(1, 130)))
        # Bytes of the rows, and the elements that the plain forms hold in 32 bits.
        if rows * (classes + pad) > (1.2e8 if dtype == "bf16" else 6.0e7):
            continue
        masks, k = rng.choice(("none", "all", "line")), log_int(1, 64)
        if op == "rules":
            c = _rules("", rows, classes, dtype, pad, steps, masks, rng.choice(("none", "all", "line")),
                       rng.choice((0, log_int(1, 3000))))
            if rows * c["history"] > 2.0e6 or (c["masks"], c["bias"], c["history"]) == ("none", "none", 0):
                continue
            if c["bias"] == "line" and (rows // steps) * classes > 1.2e7:
                continue
        elif op == "top":
            c = _top("", rows, classes, k, dtype, pad, steps, masks, rng.choice((1.0, 2.0, rng.uniform(0.5, 4.0))))
        else:
            c = _distill("", rows, classes, k, rng.choice(("both", "loss", "grad")), dtype, pad, steps,
                         rng.choice((1.0, 2.0, rng.uniform(0.5, 4.0))), rng.random() < 0.7)
        del c["name"]
        return c


# ------------------------------------------------------------------- inputs

DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16}


def _logits(case, gen):
    """Rows as a recognizer gives them: a broad floor, a leading class and a
    few that resemble it."""
    rows, classes, width = case["rows"], case["classes"], case["classes"] + case["pad"]
    x = torch.empty(rows, width, dtype=DTYPE[case["dtype"]], device="cuda")
    for r in range(0, rows, 2048):
        n = min(2048, rows - r)
        part = torch.randn(n, width, generator=gen, device="cuda").mul_(1.7)
        at = torch.randint(0, classes, (n, 6), generator=gen, device="cuda")
        lift = torch.rand(n, 6, generator=gen, device="cuda") * 6.0 + 3.0
        lift[:, 0] += 5.0
        x[r:r + n] = part.scatter_(1, at, lift)
    return x[:, :classes]


def _mask_words(n, classes, gen):
    """Allowed classes as bits, 32 a word: even masks are scripts (whole words
    of a dictionary ordered by script), odd ones short alphabets at its start;
    class 0, the blank, always stands."""
    words = (classes + 31) // 32
    script = torch.rand(n, words, generator=gen, device="cuda") < 0.4
    full = torch.where(script, -1, 0).to(torch.int32)
    short = torch.zeros(n, words, dtype=torch.int32, device="cuda")
    short[:, :2] = torch.randint(-2 ** 31, 2 ** 31, (n, min(2, words)), generator=gen, device="cuda",
                                 dtype=torch.int64).to(torch.int32)
    odd = (torch.arange(n, device="cuda") % 2 == 1)[:, None]
    m = torch.where(odd, short, full)
    m[:, 0] |= 1
    return m


def _kept_steps(case):
    """Steps of each line that carry a target; the others are padding."""
    steps = case["steps"]
    lines = case["rows"] // steps
    return [steps - (steps // 5) * (i % 3) // 2 for i in range(lines)]


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1000003 * seed + 17)
    rows, classes, steps = case["rows"], case["classes"], case["steps"]
    d = {"logits": _logits(case, gen)}
    if case["op"] == "distill":
        # The teacher's rows, kept as their best classes and the rest.
        k = min(case["k"], classes)
        values = torch.empty(rows, case["k"], device="cuda").fill_(-INF)
        indices = torch.full((rows, case["k"]), -1, dtype=torch.int32, device="cuda")
        rest = torch.empty(rows, device="cuda")
        for r in range(0, rows, 2048):
            n = min(2048, rows - r)
            t = d["logits"][r:r + n].float() + torch.randn(n, classes, generator=gen, device="cuda")
            v, i = torch.topk(t, k)
            values[r:r + n, :k], indices[r:r + n, :k] = v, i.to(torch.int32)
            rest[r:r + n] = torch.logsumexp(t.scatter_(1, i, -INF) / case["tau"], 1)
        kept = torch.tensor(_kept_steps(case), device="cuda")
        row = torch.arange(rows, device="cuda")
        indices[row % steps >= kept[row // steps]] = -1
        d.update(values=values, indices=indices, rest=rest if case["rest"] else None)
        d["grad_loss"] = torch.rand(rows, generator=gen, device="cuda") + 0.5
        return d
    lines = rows // steps
    line = (torch.arange(rows, device="cuda") // steps).to(torch.int32)
    d["masks"] = d["row_mask"] = d["bias"] = d["row_bias"] = d["history"] = None
    if case["masks"] != "none":
        d["masks"] = _mask_words(1 if case["masks"] == "all" else lines, classes, gen)
        d["row_mask"] = line if case["masks"] == "line" else torch.zeros_like(line)
    if case["bias"] != "none":
        n = 1 if case["bias"] == "all" else lines
        d["bias"] = torch.randn(n, classes, generator=gen, device="cuda")
        d["row_bias"] = line if case["bias"] == "line" else torch.zeros_like(line)
    if case["history"]:
        # Histories of every length, the first the longest, back to back; text
        # repeats its classes.
        lengths = torch.randint(0, case["history"] + 1, (rows,), generator=gen, device="cuda")
        lengths[0] = case["history"]
        offsets = torch.zeros(rows + 1, dtype=torch.int64, device="cuda")
        offsets[1:] = torch.cumsum(lengths, 0)
        u = torch.rand(int(offsets[-1]), generator=gen, device="cuda")
        d["history"] = (u * u * u * classes).to(torch.int32).clamp_(0, classes - 1)
        d["offsets"] = offsets
        d["repetition"] = torch.rand(rows, generator=gen, device="cuda") * 0.5 + 1.0
        d["frequency"] = torch.rand(rows, generator=gen, device="cuda")
        d["presence"] = torch.rand(rows, generator=gen, device="cuda")
    return d


def _gpu():
    if "gpu" not in _kept:
        sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent.parent / "ppocr-rs_amd"))
        import ppocr_hip

        _kept["hip"], _kept["gpu"] = ppocr_hip, ppocr_hip.Gpu(0)
    return _kept["hip"], _kept["gpu"]


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if case["op"] == "distill" and case["mode"] == "grad":
        # What the forward pass left for the backward pass.
        state["state"] = torch.empty(case["rows"], 4, device="cuda")
        for r in range(0, case["rows"], 2048):
            part = slice(r, min(r + 2048, case["rows"]))
            state["state"][part] = _distill_sums(state, case, part)[0].float()
    if own:
        hip, state["gpu"] = _gpu()
        if case["op"] == "distill":
            state["teacher"] = hip.TopLogits(state["values"], state["indices"], state["rest"])
        else:
            state["rules"] = None
            if any(state[k] is not None for k in ("masks", "bias", "history")):
                kw = {k: state[k] for k in ("masks", "row_mask", "bias", "row_bias")}
                if state["history"] is not None:
                    kw.update(history=state["history"], history_offsets=state["offsets"],
                              repetition=state["repetition"], frequency=state["frequency"],
                              presence=state["presence"])
                state["rules"] = hip.LogitRules(case["classes"], **kw)
    return state


# --------------------------------------------------------------- plain forms

def _allowed(masks, row_mask, classes):
    shift = torch.arange(32, device="cuda", dtype=torch.int32)
    bits = (masks[:, :, None] >> shift & 1).reshape(masks.shape[0], -1)[:, :classes] != 0
    return bits[row_mask.long()]


def _apply_rules(s, case):
    x = s["logits"].float()
    if s["history"] is not None:
        rows, classes = x.shape
        at = torch.arange(s["history"].shape[0], device="cuda")
        row = torch.searchsorted(s["offsets"], at, right=True) - 1
        n = torch.zeros(rows * classes, device="cuda")
        n.scatter_add_(0, row * classes + s["history"].long(), torch.ones(at.shape[0], device="cuda"))
        n = n.reshape(rows, classes)
        r = s["repetition"][:, None]
        y = torch.where(x > 0, x / r, x * r) - (s["frequency"][:, None] * n + s["presence"][:, None])
        x = torch.where(n > 0, y, x)
    if s["bias"] is not None:
        x = x + s["bias"][s["row_bias"].long()]
    if s["masks"] is not None:
        x = torch.where(_allowed(s["masks"], s["row_mask"], case["classes"]), x, -INF)
    return x


def _plain_top(s, case):
    """Best classes by one 64-bit key a class: the value's order above, the
    lower class first below."""
    x = _apply_rules(s, case) + 0.0
    rows, classes = x.shape
    k = case["k"]
    bits = x.view(torch.int32).long()
    order = torch.where(bits >= 0, bits, -2147483648 - bits)
    key = order * 4294967296 + (classes - 1 - torch.arange(classes, device="cuda"))
    best = torch.topk(key, min(k, classes), 1).values
    index = classes - 1 - (best & 4294967295)
    value = torch.gather(x, 1, index)
    y = (x / case["tau"]).scatter_(1, index, -INF)
    top = y.max(1, keepdim=True).values
    rest = torch.log(torch.exp(y - torch.where(top == -INF, 0.0, top)).sum(1)) + top[:, 0]
    values = torch.full((rows, k), -INF, device="cuda")
    indices = torch.full((rows, k), -1, dtype=torch.int32, device="cuda")
    values[:, :value.shape[1]] = value
    indices[:, :value.shape[1]] = torch.where(value == -INF, -1, index).to(torch.int32)
    return {"values": values, "indices": indices, "rest": rest}


def _distill_sums(s, case, part=slice(None)):
    """Maximum and sum of exp over all classes and over those that are no
    entry of the teacher's (each sum relative to its own maximum).  The sums
    are long and the loss takes a difference of their logs that nearly cancels,
    so they are held in 64 bits, the whole as the rest plus the entries."""
    x = s["logits"][part].float()
    index = s["indices"][part].long()
    target = (index >= 0).any(1)
    at = torch.where(index >= 0, index, index.max(1, keepdim=True).values.clamp_min(0))
    y = x.scatter(1, at, -INF)
    m, mr = x.max(1, keepdim=True).values, y.max(1, keepdim=True).values
    low = torch.where(mr == -INF, 0.0, mr)
    zr = torch.exp((y - low) / case["tau"]).sum(1, dtype=torch.float64)
    entry = torch.gather(x, 1, index.clamp_min(0)).double()
    entry = torch.where(index >= 0, torch.exp((entry - m) / case["tau"]), 0.0).sum(1)
    z = entry + zr * torch.exp((low.double() - m)[:, 0] / case["tau"])
    sums = torch.stack([m[:, 0].double(), z, mr[:, 0].double(), zr], 1)
    return torch.where(target[:, None], sums, 0.0), x, index, target


def _teacher(s, case):
    """The teacher's share of each entry and of the rest, and their logs, in
    64 bits: the loss is a difference of logs that nearly cancel."""
    t = torch.where(s["indices"] >= 0, s["values"].double() / case["tau"], -INF)
    rest = torch.full((case["rows"],), -INF, device="cuda") if s["rest"] is None else s["rest"]
    t = torch.cat([t, rest.double()[:, None]], 1)
    t = t - t.max(1, keepdim=True).values
    logq = t - torch.log(torch.exp(t).sum(1, keepdim=True))
    return torch.exp(logq), logq


def _plain_distill(s, case):
    tau = case["tau"]
    q, logq = _teacher(s, case)
    if case["mode"] == "grad":
        x = s["logits"].float()
        index = s["indices"].long()
        target, sums = (index >= 0).any(1), s["state"]
    else:
        sums, x, index, target = _distill_sums(s, case)
    out = {}
    if case["mode"] != "grad":
        m, z, mr, zr = (sums[:, i:i + 1] for i in range(4))
        entry = torch.gather(x, 1, index.clamp_min(0))
        logp = torch.cat([(entry - m) / tau, (mr - m) / tau + torch.log(zr)], 1) - torch.log(z)
        loss = torch.where(q > 0, q * (logq - logp), 0.0).sum(1) * (tau * tau)
        out["loss"] = torch.where(target, loss, 0.0).float()
        if case["mode"] == "loss":
            out["state"] = sums.float()
            return out
    q = q.float()
    m, z, mr, zr = (sums[:, i:i + 1].float() for i in range(4))
    scale = s["grad_loss"][:, None] * tau
    p = torch.exp((x - m) / tau) / z
    share = torch.where(zr > 0, q[:, -1:] * torch.exp((m - mr) / tau) * z / zr, 0.0)
    grad = p * (1.0 - share)
    at = torch.where(index >= 0, index, index.max(1, keepdim=True).values.clamp_min(0))
    # Places without an entry repeat one of their row's.
    first = index.argmax(1, keepdim=True)
    entry = torch.gather(p, 1, at) - torch.where(index >= 0, q[:, :-1], torch.gather(q, 1, first))
    grad.scatter_(1, at, entry)
    grad = torch.where(target[:, None], grad * scale, 0.0)
    out["grad"] = grad.to(s["logits"].dtype)
    return out


def run(state):
    s, case = state, state["case"]
    if not own:
        if case["op"] == "rules":
            return _apply_rules(s, case).to(s["logits"].dtype)
        return _plain_top(s, case) if case["op"] == "top" else _plain_distill(s, case)
    gpu = s["gpu"]
    if case["op"] == "rules":
        return gpu.logit_rules(s["logits"], s["rules"])
    if case["op"] == "top":
        top = gpu.top_logits(s["logits"], case["k"], s["rules"], case["tau"])
        return {"values": top.values, "indices": top.indices, "rest": top.rest}
    if case["mode"] == "loss":
        loss, sums = gpu.distill_loss(s["logits"], s["teacher"], case["tau"])
        return {"loss": loss, "state": sums}
    if case["mode"] == "grad":
        return {"grad": gpu.distill_grad(s["logits"], s["teacher"], s["state"], case["tau"], s["grad_loss"])}
    loss, grad = gpu.distill(s["logits"], s["teacher"], case["tau"], s["grad_loss"])
    return {"loss": loss, "grad": grad}


# -------------------------------------------------------------------- work

def work(case):
    rows, classes = case["rows"], case["classes"]
    es = 4 if case["dtype"] == "f32" else 2
    n = float(rows) * classes
    lines = rows // case["steps"]
    if case["op"] == "distill":
        k = case["k"]
        live = float(sum(_kept_steps(case)))
        read = live * classes * es + rows * k * 4.0 + live * (k * 4 + (4 if case["rest"] else 0))
        written = {"loss": rows * 20.0, "grad": n * es, "both": n * es + rows * 4.0}[case["mode"]]
        if case["mode"] == "grad":
            read += live * 16.0
        if case["mode"] != "loss":
            read += live * 4.0
        return {"bytes": read + written, "flops": live * classes * (8.0 if case["mode"] == "both" else 5.0)}
    read = n * es
    if case["masks"] != "none":
        read += (1 if case["masks"] == "all" else lines) * classes / 8.0 + rows * 4.0
    if case["bias"] != "none":
        read += (1 if case["bias"] == "all" else lines) * classes * 4.0 + rows * 4.0
    if case["history"]:
        read += rows * (case["history"] / 2.0 * 4.0 + 20.0)
    written = n * es if case["op"] == "rules" else rows * (8.0 * case["k"] + 4.0)
    return {"bytes": read + written, "flops": n * (2.0 if case["op"] == "rules" else 5.0)}


# ------------------------------------------------------------------- exact

def _exact_rules(d, case):
    """Row blocks in 64 bits: every class's count by a histogram of its row's
    history, the masks' bits one class at a time."""
    classes = case["classes"]
    c = torch.arange(classes, device="cuda")
    step = max(1, 40_000_000 // classes)
    for a in range(0, case["rows"], step):
        b = min(a + step, case["rows"])
        x = d["logits"][a:b].double()
        if d["history"] is not None:
            lo, hi = int(d["offsets"][a]), int(d["offsets"][b])
            lengths = d["offsets"][a + 1:b + 1] - d["offsets"][a:b]
            row = torch.repeat_interleave(torch.arange(b - a, device="cuda"), lengths)
            n = torch.bincount(row * classes + d["history"][lo:hi].long(), minlength=(b - a) * classes)
            n = n.reshape(b - a, classes).double()
            r, f, p = (d[k][a:b, None].double() for k in ("repetition", "frequency", "presence"))
            seen = n > 0
            x = torch.where(seen & (x > 0), x / r, torch.where(seen, x * r, x))
            x = x - seen * (f * n + p)
        if d["bias"] is not None:
            x = x + d["bias"].double()[d["row_bias"][a:b].long()]
        if d["masks"] is not None:
            word = d["masks"][:, c // 32].long()[d["row_mask"][a:b].long()]
            x[(word >> (c % 32)) % 2 == 0] = -INF
        yield a, b, x


def _exact_top(d, case):
    rows, k, tau = case["rows"], case["k"], case["tau"]
    values = torch.full((rows, k), -INF, dtype=torch.float64, device="cuda")
    indices = torch.full((rows, k), -1, dtype=torch.int32, device="cuda")
    rest = torch.empty(rows, dtype=torch.float64, device="cuda")
    for a, b, x in _exact_rules(d, case):
        v, i = torch.sort(x, dim=1, descending=True, stable=True)
        n = min(k, case["classes"])
        values[a:b, :n] = v[:, :n]
        indices[a:b, :n] = torch.where(v[:, :n] == -INF, -1, i[:, :n]).to(torch.int32)
        rest[a:b] = torch.logsumexp(v[:, n:] / tau, 1) if n < case["classes"] else -INF
    return {"values": values, "indices": indices, "rest": rest}


def _exact_distill(d, case):
    rows, classes, tau = case["rows"], case["classes"], case["tau"]
    want = {"loss": [], "state": [], "grad": []}
    step = max(1, 20_000_000 // classes)
    for a in range(0, rows, step):
        b = min(a + step, rows)
        x = d["logits"][a:b].double()
        index, valid = d["indices"][a:b].long(), d["indices"][a:b] >= 0
        target = valid.any(1)
        # Entries as a dense table; classes of the rest share one bucket.
        t = torch.full((b - a, classes + 1), -INF, dtype=torch.float64, device="cuda")
        t.scatter_(1, torch.where(valid, index, classes), d["values"][a:b].double())
        t = t[:, :classes]
        entry = t > -INF
        bucket = d["rest"][a:b].double() if d["rest"] is not None else torch.full_like(t[:, 0], -INF)
        total = torch.logaddexp(torch.logsumexp(t / tau, 1), bucket)
        logq, logq0 = t / tau - total[:, None], bucket - total
        logp = torch.log_softmax(x / tau, 1)
        logp0 = torch.logsumexp(torch.where(entry, -INF, logp), 1)
        loss = torch.where(entry, torch.exp(logq) * (logq - logp), 0.0).sum(1)
        loss = loss + torch.where(logq0 > -INF, torch.exp(logq0) * (logq0 - logp0), 0.0)
        want["loss"].append(torch.where(target, loss * tau * tau, 0.0))
        if case["mode"] == "loss":
            y = torch.where(entry, -INF, x)
            m, mr = x.amax(1), y.amax(1)
            sums = torch.stack([m, torch.exp(torch.logsumexp(x / tau, 1) - m / tau), mr,
                                torch.where(mr > -INF, torch.exp(torch.logsumexp(y / tau, 1) - mr / tau), 0.0)], 1)
            want["state"].append(torch.where(target[:, None], sums, 0.0))
        else:
            p = torch.exp(logp)
            other = torch.where(logq0 > -INF, torch.exp(logq0 - logp0), 0.0)[:, None] * p
            g = (p - torch.where(entry, torch.exp(logq), other)) * tau * d["grad_loss"][a:b, None].double()
            want["grad"].append(torch.where(target[:, None], g, 0.0))
    keys = {"loss": ("loss", "state"), "grad": ("grad",), "both": ("loss", "grad")}[case["mode"]]
    return {k: torch.cat(want[k]) for k in keys}


def exact(case, seed):
    d = _inputs(case, seed)
    if case["op"] == "rules":
        return torch.cat([x for _, _, x in _exact_rules(d, case)])
    return _exact_top(d, case) if case["op"] == "top" else _exact_distill(d, case)


if __name__ == "__main__":
    rng = random.Random(7)
    for c in listed() + [draw(rng) for _ in range(6)]:
        print(c, work(c))
