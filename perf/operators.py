"""The training losses of large classifiers, as they are measured: cross entropy of a linear head over many classes
without its logits being kept, and distillation from a teacher's top logits; each alone or with its gradients."""
import math

import torch

if torch.cuda.is_available():
    DEVICE = "cuda"
else:
    DEVICE = "cpu"

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def head(name, rows, classes, dim, dtype, grad=True, scale=1.0, smoothing=0.0, ignored=0.0):
    return {"name": name, "op": "linear_cross_entropy", "rows": rows, "classes": classes, "dim": dim, "dtype": dtype,
            "grad": grad, "scale": scale, "smoothing": smoothing, "ignored": ignored}


def distil(name, rows, classes, top, dtype, grad=True, temperature=2.0, tail=False):
    return {"name": name, "op": "distill_topk", "rows": rows, "classes": classes, "top": top, "dtype": dtype,
            "grad": grad, "temperature": temperature, "tail": tail}


def listed():
    return [
        # one crop scored against a small gallery: nothing but latency
        head("head 1x1000", 1, 1000, 128, "fp32", grad=False),
        # one short training step of an identity head on normalised embeddings, whole in 32 bits
        head("head 61x10007 fp32", 61, 10007, 512, "fp32", scale=32.0),
        # the step of one GPU on a large identity head: the weight and its gradient are what is moved
        head("head 256x1000003", 256, 1000003, 512, "bf16", scale=32.0),
        # ordinary fine-tuning, odd sizes, padded rows and smoothed labels
        head("head 2039x50021 fp16", 2039, 50021, 768, "fp16", smoothing=0.1, ignored=0.25),
        # scoring held-out text: the value alone
        head("head 4096x32000 value", 4096, 32000, 4096, "bf16", grad=False, ignored=0.05),
        # the largest step: a long batch over a large vocabulary
        head("head 8192x131072", 8192, 131072, 2048, "bf16", ignored=0.05),
        # one row: latency again
        distil("distil 1x32000", 1, 32000, 16, "bf16"),
        # the class columns of four 640x640 images' anchors: very many rows of two classes
        distil("distil 408000x2 fp32", 408000, 2, 2, "fp32"),
        # ordinary, odd rows that start off any boundary, the teacher's other classes as one
        distil("distil 1021x50021 fp16 tail", 1021, 50021, 32, "fp16", tail=True),
        # the value alone over a held-out batch
        distil("distil 2048x32000 value", 2048, 32000, 20, "bf16", grad=False, temperature=1.0),
        # long batches over a large vocabulary
        distil("distil 8192x131072", 8192, 131072, 64, "bf16", tail=True),
        distil("distil 3001x100003 fp32", 3001, 100003, 100, "fp32", temperature=1.0),
    ]


def spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    dtype = rng.choice(sorted(TYPES))
    if rng.random() < 0.5:
        while True:
            c = head("", spread(rng, 1, 8192), spread(rng, 2, 1000000), spread(rng, 16, 4096), dtype,
                     grad=rng.random() < 0.75, scale=rng.choice([1.0, 1.0, 16.0, 32.0]),
                     smoothing=rng.choice([0.0, 0.0, 0.1]), ignored=rng.choice([0.0, 0.1, 0.5]))
            most = 2 ** 30 if dtype == "fp32" else 2 ** 32
            if c["rows"] * c["classes"] <= 2 ** 30 and c["rows"] * c["classes"] * c["dim"] <= 512 * most \
                    and c["classes"] * c["dim"] <= 2 ** 29:
                break
    else:
        while True:
            classes = spread(rng, 2, 262144)
            c = distil("", spread(rng, 1, 500000), classes, spread(rng, 1, min(classes, 256)), dtype,
                       grad=rng.random() < 0.75, temperature=rng.choice([1.0, 2.0, 4.0]), tail=rng.random() < 0.4)
            if c["rows"] * classes * SIZE[dtype] <= 2 ** 31:
                break
    del c["name"]
    return c


def upstream(case):
    """What comes down to each row's loss: nothing given (the mean over the rows), or in 16 bits of short range a scaled one,
    as such a training run has it."""
    if case["dtype"] != "fp16" or not case["grad"]:
        return None
    return torch.full((case["rows"],), 1024.0 / math.sqrt(case["rows"]), device=DEVICE)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    n, v, dtype = case["rows"], case["classes"], TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE)

    if case["op"] == "linear_cross_entropy":
        d = case["dim"]
        label = torch.randint(0, v, (n,), generator=g, device=DEVICE)
        weight = normal(v, d)
        if case["scale"] != 1.0:                      # embeddings on the unit sphere, near their class
            weight /= weight.norm(dim=1, keepdim=True)
            hidden = normal(n, d) / math.sqrt(d) + 0.4 * weight[label]
            hidden /= hidden.norm(dim=1, keepdim=True)
        else:                                         # logits of a deviation of about two, the label's raised
            weight *= 2.0 / math.sqrt(d)
            hidden = normal(n, d) + 1.5 * weight[label]
        padded = torch.rand(n, generator=g, device=DEVICE) < case["ignored"]
        label = torch.where(padded, torch.full_like(label, -100), label)
        return {"case": case, "hidden": hidden.to(dtype), "weight": weight.to(dtype), "label": label,
                "grad_loss": upstream(case)}
    logits = normal(n, v).mul_(2.0).to(dtype)
    teacher = normal(n, v).add_(logits)
    values, index = teacher.topk(case["top"], dim=1)
    state = {"case": case, "logits": logits, "values": values, "index": index, "lse": None,
             "grad_loss": upstream(case)}
    if case["tail"]:                                  # of all the teacher's logits, at the temperature
        state["lse"] = teacher.div_(case["temperature"]).logsumexp(dim=1)
    return state


def plain_head(hidden, weight, label, scale, smoothing, grad, grad_loss):
    n, v = hidden.shape[0], weight.shape[0]
    h, w = hidden.float(), weight.float()
    z = torch.matmul(h, w.t()) * scale
    counted = (label >= 0)[:, None]
    at = label.clamp(min=0)[:, None]
    z_label = z.gather(1, at)
    top = z.amax(dim=1, keepdim=True)
    e = torch.exp(z - top)
    lse = top + e.sum(dim=1, keepdim=True).log()
    # the label's class stays out of the sum: a sure row's loss and gradient are what the others leave
    others = e.scatter(1, at, 0.0).sum(dim=1, keepdim=True)
    nll = torch.where(z_label < top, lse - z_label, torch.log1p(others))
    loss = (1.0 - smoothing) * nll + smoothing * (lse - z.mean(dim=1, keepdim=True))
    loss = torch.where(counted, loss, torch.zeros_like(loss))[:, 0]
    if not grad:
        return loss
    p = torch.exp(z - lse) - smoothing / v
    p.scatter_(1, at, torch.expm1(-nll) + (smoothing - smoothing / v))
    p = torch.where(counted, p, torch.zeros_like(lse)) * scale
    p = p * (1.0 / n if grad_loss is None else grad_loss[:, None])
    return loss, torch.matmul(p, w).to(hidden.dtype), torch.matmul(p.t(), h).to(weight.dtype)


def plain_distil(logits, values, index, temperature, tail_lse, grad, grad_loss):
    n = logits.shape[0]
    u = logits.float() / temperature
    top = u.amax(dim=1, keepdim=True)
    e = torch.exp(u - top)
    # the loss is a difference of logarithms far larger than itself: sums and what is one value a teacher's entry are in 64 bits
    total = e.sum(dim=1, keepdim=True, dtype=torch.float64)
    logp = u.gather(1, index).double() - top.double() - total.log()
    t = values.double() / temperature
    if tail_lse is None:
        t_top = t.amax(dim=1, keepdim=True)
        logq = t - (t_top + torch.exp(t - t_top).sum(dim=1, keepdim=True).log())
    else:
        logq = t - tail_lse.double()[:, None]
    q = torch.exp(logq)
    sum_q = q.sum(dim=1, keepdim=True)
    loss = (q * (logq - logp)).sum(dim=1, keepdim=True)
    outside = None
    if tail_lse is not None and index.shape[1] < logits.shape[1]:
        outside = torch.ones_like(e).scatter_(1, index, 0.0)
        rest_q = (1.0 - sum_q).clamp(min=0.0)
        rest_p = (e * outside).sum(dim=1, keepdim=True, dtype=torch.float64) / total
        rest = rest_q * (torch.log(rest_q) - torch.log(rest_p))
        loss = loss + torch.where(rest_q > 0, rest, torch.zeros_like(rest))
    loss = (loss[:, 0] * temperature ** 2).float()
    if not grad:
        return loss
    if outside is not None:
        factor = (sum_q + rest_q).float() - outside * (rest_q / rest_p).float()
    else:
        factor = sum_q.float()
    d = (e / total.float()) * factor
    d.scatter_add_(1, index, -q.float())
    d = d * (temperature / n if grad_loss is None else temperature * grad_loss[:, None])
    return loss, d.to(logits.dtype)


def run(state):
    case = state["case"]
    if case["op"] == "linear_cross_entropy":
        if own:
            from face_detection_amd import linear_cross_entropy_batch
            return linear_cross_entropy_batch(state["hidden"], state["weight"], state["label"], logit_scale=case["scale"],
                                              label_smoothing=case["smoothing"], grad_loss=state["grad_loss"],
                                              return_grad=case["grad"])
        return plain_head(state["hidden"], state["weight"], state["label"], case["scale"], case["smoothing"], case["grad"],
                          state["grad_loss"])
    if own:
        from face_detection_amd import distill_topk_batch
        return distill_topk_batch(state["logits"], state["values"], state["index"], temperature=case["temperature"],
                                  teacher_lse=state["lse"], grad_loss=state["grad_loss"], return_grad=case["grad"])
    return plain_distil(state["logits"], state["values"], state["index"], case["temperature"], state["lse"], case["grad"],
                        state["grad_loss"])


def work(case):
    n, v, size = case["rows"], case["classes"], SIZE[case["dtype"]]
    if case["op"] == "linear_cross_entropy":
        inputs = (n + v) * case["dim"] * size
        ways = 3 if case["grad"] else 1
        return {"bytes": inputs * (2 if case["grad"] else 1) + n * 12, "flops": ways * 2 * n * v * case["dim"] + 4 * n * v}
    each = n * v * size
    return {"bytes": each * (2 if case["grad"] else 1) + n * case["top"] * 12 + n * (8 if case["tail"] else 4),
            "flops": (6 if case["grad"] else 4) * n * v + 8 * n * case["top"]}


def exact(case, seed):
    """From the definitions, in 64 bits, some rows at a time."""
    state = prepare(case, seed)
    n, v = case["rows"], case["classes"]
    step = max(1, 2 ** 28 // v)
    down = upstream(case)
    down = torch.full((n, 1), 1.0 / n, dtype=torch.float64, device=DEVICE) if down is None else down.double()[:, None]
    losses, parts = [], []
    if case["op"] == "linear_cross_entropy":
        w = state["weight"].double()
        grad_w = torch.zeros_like(w) if case["grad"] else None
        eps = case["smoothing"]
        for a in range(0, n, step):
            h, label = state["hidden"][a:a + step].double(), state["label"][a:a + step]
            logp = torch.log_softmax(case["scale"] * torch.mm(h, w.t()), dim=1)
            target = torch.full_like(logp, eps / v)
            rows = torch.arange(len(h), device=h.device)
            target[rows, label.clamp(min=0)] += 1.0 - eps
            counted = (label >= 0).double()
            losses.append(-(target * logp).sum(1) * counted)
            if case["grad"]:
                delta = (logp.exp_() - target) * (counted[:, None] * case["scale"] * down[a:a + step])
                parts.append(torch.mm(delta, w))
                grad_w += torch.mm(delta.t().contiguous(), h)
        loss = torch.cat(losses)
        return (loss, torch.cat(parts), grad_w) if case["grad"] else loss
    tau = case["temperature"]
    for a in range(0, n, step):
        logp = torch.log_softmax(state["logits"][a:a + step].double() / tau, dim=1)
        t, index = state["values"][a:a + step].double() / tau, state["index"][a:a + step]
        whole = torch.logsumexp(t, 1) if state["lse"] is None else state["lse"][a:a + step].double()
        q = torch.exp(t - whole[:, None])
        kl = (torch.special.xlogy(q, q) - q * logp.gather(1, index)).sum(1)
        p = logp.exp()
        away = torch.zeros_like(p).scatter_(1, index, q)       # q where the teacher has one
        scale = q.sum(1, keepdim=True)
        delta = p * scale - away
        if case["tail"] and case["top"] < v:
            rest_q = (1 - scale).clamp(min=0)
            other = p.scatter(1, index, 0.0)
            rest_p = other.sum(1, keepdim=True)
            kl += (torch.special.xlogy(rest_q, rest_q) - torch.special.xlogy(rest_q, rest_p))[:, 0]
            delta = p * (scale + rest_q) - away - other * (rest_q / rest_p)
        losses.append(tau ** 2 * kl)
        if case["grad"]:
            parts.append(delta * (tau * down[a:a + step]))
    return (torch.cat(losses), torch.cat(parts)) if case["grad"] else torch.cat(losses)
