"""Timed cases of what lies between a hidden state and the sampler when every request
has something of its own: the projection shared by all rows with a low-rank adapter
for each row's request, its gradients, and the rules on a row's logits (penalties for
repeated tokens, biases, a grammar's mask).

A pass is one call of a serving or training program: the projection of a batch of
hidden states, the projection forward and backward, or the rules of one decode step.
Where ``own`` is false the same mathematics is written with elementary torch operations.

Definitions (in float32 or wider, one rounding at the end):

  project   u[n] = s_a * A_a h[n], out[n] = W h[n] + B_a u[n] with a = adapter[n];
            W h[n] alone where a is outside [0, adapters)
  gradients du[n] = s_a * B_a^T dout[n], dh[n] = W^T dout[n] + A_a^T du[n],
            dA_a = sum of du[n] h[n]^T, dB_a = sum of dout[n] u[n]^T over the rows n of adapter a
  rules     v = c * tanh(logit / c) (the logit itself without a softcap);
            a token of the row's history: v > 0 ? v / r : v * r;
            one that the history holds k > 0 times behind its prompt: v - f * k - p;
            one with a bias: v + b (of several entries for a token the last counts);
            one that the row's mask does not allow: -infinity. A row that may answer
            with nothing is flagged.
"""
import math

import torch

own = False


def listed():
    return [
        # One token of one request with its adapter: the weights are read once, latency counts.
        dict(name="project_1", kind="project", rows=1, dim=2816, out=262144, rank=16, adapters=4, dtype="bf16", odtype="f32"),
        # A few tokens through a small inner projection: the call itself is what it costs.
        dict(name="project_5_small", kind="project", rows=5, dim=640, out=2560, rank=8, adapters=3, dtype="bf16", odtype="bf16"),
        # A decode step of 64 requests over 24 adapters.
        dict(name="project_64", kind="project", rows=64, dim=2816, out=262144, rank=16, adapters=24, dtype="bf16", odtype="bf16"),
        # Odd sizes in float32.
        dict(name="project_97_f32", kind="project", rows=97, dim=1000, out=50257, rank=12, adapters=7, dtype="f32", odtype="f32"),
        # The logits of every position of several prompts.
        dict(name="project_4096", kind="project", rows=4096, dim=2816, out=262144, rank=32, adapters=9, dtype="bf16", odtype="bf16"),
        # A training step of three adapters beside a small model's odd vocabulary.
        dict(name="train_1021", kind="train", rows=1021, dim=1152, out=32003, rank=8, adapters=3, dtype="bf16", odtype="bf16"),
        # The same in float32.
        dict(name="train_300_f32", kind="train", rows=300, dim=768, out=8192, rank=16, adapters=2, dtype="f32", odtype="f32"),
        # A large batch through a wide inner projection.
        dict(name="train_8192", kind="train", rows=8192, dim=2816, out=11264, rank=64, adapters=5, dtype="bf16", odtype="bf16"),
        # One session's decode step, in place: a few hundred tokens of its history change.
        dict(name="rules_1", kind="rules", rows=1, vocab=262144, dtype="bf16", to="inplace", cap=0.0, history=700, bias=8, mask="none", per_row=False),
        # Structured answers: each of 64 rows has a grammar that allows few tokens.
        dict(name="rules_grammar_64", kind="rules", rows=64, vocab=262144, dtype="bf16", to="inplace", cap=0.0, history=300, bias=0, mask="few", per_row=True),
        # An odd vocabulary in float32, long histories, masks that allow most tokens.
        dict(name="rules_9_f32", kind="rules", rows=9, vocab=50257, dtype="f32", to="f32", cap=0.0, history=60000, bias=300, mask="most", per_row=False),
        # The largest decode step: softcap, penalties, biases and masks of 512 rows.
        dict(name="rules_512", kind="rules", rows=512, vocab=262144, dtype="bf16", to="f32", cap=30.0, history=2000, bias=50, mask="most", per_row=True),
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("project", "project", "train", "train", "rules", "rules", "rules"))
    c = dict(kind=kind, dtype=rng.choice(("bf16", "bf16", "f32")))
    if kind == "rules":
        c["rows"] = _spread(rng, 1, 512)
        c["vocab"] = 262144 if rng.random() < 0.3 else _spread(rng, 8000, 262144)
        c["to"] = rng.choice(("inplace", "inplace", "f32", "same"))
        c["cap"] = rng.choice((0.0, 0.0, 30.0))
        c["history"] = _spread(rng, 1, 60000 if c["rows"] <= 16 else 4000)
        c["bias"] = rng.choice((0, _spread(rng, 1, 300)))
        c["mask"] = rng.choice(("none", "few", "most"))
        c["per_row"] = rng.random() < 0.5
        return c
    c["rows"] = _spread(rng, 1, 4096 if kind == "project" else 8192)
    c["dim"] = _spread(rng, 256, 2816)
    if rng.random() < 0.8:  # models' widths are round, with few exceptions
        c["dim"] = max(256, c["dim"] - c["dim"] % 64)
    c["out"] = _spread(rng, 1000, 262144 if kind == "project" else 32768)
    if c["dtype"] == "f32":  # float32 layers are small ones
        c["rows"], c["out"] = min(c["rows"], 1024), min(c["out"], 65536)
    c["rank"] = rng.choice((4, 8, 8, 16, 16, 32, 64, _spread(rng, 1, 64)))
    c["adapters"] = _spread(rng, 1, 32 if kind == "project" else 8)
    c["odtype"] = "f32" if c["dtype"] == "f32" else rng.choice(("bf16", "f32"))
    return c


DTYPES = dict(f32=torch.float32, bf16=torch.bfloat16)
ALLOWED = dict(few=0.002, most=0.97)  # share of the vocabulary that a mask allows
PENALTIES = dict(repetition_penalty=1.1, presence_penalty=0.4, frequency_penalty=0.15)
EMPTY = 1  # flag of a row that may answer with nothing


def _gen(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)


def _rand(gen, *shape):
    return torch.rand(*shape, generator=gen, device="cuda")


def _inputs(c, seed):
    return _rules_inputs(c, seed) if c["kind"] == "rules" else _project_inputs(c, seed)


def _project_inputs(c, seed):
    gen, dt = _gen(seed), DTYPES[c["dtype"]]
    n, d, v, r, k = c["rows"], c["dim"], c["out"], c["rank"], c["adapters"]
    s = dict(h=_randn(gen, n, d).to(dt), w=(_randn(gen, v, d, dtype=dt) * (3.0 / math.sqrt(d))).to(dt))
    # adapters as training leaves them: an update a tenth as large as what the weights give
    s["a"] = (_randn(gen, k, r, d) / math.sqrt(d)).to(dt)
    s["b"] = (_randn(gen, k, v, r, dtype=dt) * (0.15 / math.sqrt(r))).to(dt)
    s["scale"] = 1.0 + _rand(gen, k)
    # Tokens of a request lie together; every ninth request has no adapter.
    runs = 1 if n <= 64 else n // 40
    ids = torch.randint(k, (n // runs + 1,), generator=gen, device="cuda")
    ids = torch.where(_rand(gen, n // runs + 1) < 1 / 9, -1, ids)
    s["adapter"] = ids.repeat_interleave(runs)[:n].int().contiguous()
    if c["kind"] == "train":
        s["dout"] = (_randn(gen, n, v, dtype=dt) / n).to(dt)
    return s


def _ragged(gen, rows, most):
    """Offsets of rows of up to `most` entries, the first as long as that."""
    n = (_rand(gen, rows) * (most + 1)).int()
    n[0] = most
    return torch.cat([torch.zeros(1, device="cuda", dtype=torch.int32), torch.cumsum(n, 0, dtype=torch.int32)])


def _rules_inputs(c, seed):
    gen, dt, n, v = _gen(seed), DTYPES[c["dtype"]], c["rows"], c["vocab"]
    s = dict(logits=(_randn(gen, n, v) * 4.0).to(dt), mask=None, mask_rows=None, bias_ids=None, bias_values=None, bias_offsets=None)
    # Words of a text: few of them make up most of it.
    s["offsets"] = _ragged(gen, n, c["history"])
    total = int(s["offsets"][-1])
    s["history"] = (v * _rand(gen, total) ** 4).int().clamp_max(v - 1)
    lengths = s["offsets"][1:] - s["offsets"][:-1]
    s["prompt"] = (lengths * _rand(gen, n)).int()
    if c["bias"]:
        s["bias_offsets"] = _ragged(gen, n, c["bias"])
        total = int(s["bias_offsets"][-1])
        s["bias_ids"] = torch.randint(v, (total,), generator=gen, device="cuda", dtype=torch.int32)
        s["bias_values"] = torch.where(_rand(gen, total) < 0.1, -math.inf, 4.0 * _randn(gen, total))  # some are bans
    if c["mask"] != "none":
        masks = max(1, n // 2)  # requests share grammars; every seventh row has none
        words = -(-v // 32)
        s["mask"] = torch.empty(masks, words, dtype=torch.int32, device="cuda")
        bit = torch.arange(32, device="cuda", dtype=torch.int32)
        for i in range(masks):
            ok = _rand(gen, words, 32) < ALLOWED[c["mask"]]
            if i == 1:  # a grammar that has come to its end
                ok[:] = False
            s["mask"][i] = (ok.int() << bit).sum(1).int()
        s["mask_rows"] = (torch.arange(n, device="cuda") % masks).int()
        s["mask_rows"][6::7] = -1
    f = _rand(gen, n, 1) if c["per_row"] else 1.0
    s["params"] = {k: (x - 1.0) * f + 1.0 if k == "repetition_penalty" else x * f for k, x in PENALTIES.items()}
    return s


def prepare(case, seed):
    c = dict(case)
    s = _inputs(c, seed)
    s["case"] = c
    if own and c["kind"] == "rules":
        from gemmaedge_amd import rules as R

        s["config"] = R.RuleConfig(softcap=c["cap"], **PENALTIES)
        s["row_params"] = None
        if c["per_row"]:  # kept on the device while the requests live
            p = {k: x[:, 0].tolist() for k, x in s["params"].items()}
            s["row_params"] = R.row_params([R.RuleConfig(softcap=c["cap"], **{k: x[i] for k, x in p.items()}) for i in range(c["rows"])])
    elif own:
        from gemmaedge_amd import projection as P

        s["projection"] = P.Projection(c["rows"], c["dim"], c["out"], max_rank=c["rank"], max_adapters=c["adapters"],
                                       dtype=DTYPES[c["dtype"]], train=c["kind"] == "train")
    return s


# ---- plain forms --------------------------------------------------------------


def _project(s, c):
    h = s["h"].float()
    y = h @ s["w"].float().t()
    for k in range(c["adapters"]):
        rows = torch.nonzero(s["adapter"] == k)[:, 0]
        u = (h[rows] @ s["a"][k].float().t()) * s["scale"][k]
        y[rows] += u @ s["b"][k].float().t()
    return y.to(DTYPES[c["odtype"]])


def _project_backward(s, c):
    h, g = s["h"].float(), s["dout"].float()
    dh = g @ s["w"].float()
    da, db = torch.zeros_like(s["a"]), torch.zeros_like(s["b"])
    for k in range(c["adapters"]):
        rows = torch.nonzero(s["adapter"] == k)[:, 0]
        a, b, scale = s["a"][k].float(), s["b"][k].float(), s["scale"][k]
        u = (h[rows] @ a.t()) * scale
        du = (g[rows] @ b) * scale
        dh[rows] += du @ a
        da[k] = (du.t() @ h[rows]).to(da.dtype)
        db[k] = (g[rows].t() @ u).to(db.dtype)
    return dh.to(s["h"].dtype), da, db


def _row_of(offsets, total):
    return torch.bucketize(torch.arange(total, device="cuda", dtype=torch.int32), offsets[1:], right=True)


def _rules(s, c):
    n, v = c["rows"], c["vocab"]
    x = s["logits"].float()
    if c["cap"] > 0:
        x = c["cap"] * torch.tanh(x / c["cap"])
    p = s["params"]
    row = _row_of(s["offsets"], s["history"].numel())
    at = row * v + s["history"].long()
    behind = torch.arange(s["history"].numel(), device="cuda") - s["offsets"][row] >= s["prompt"][row]
    seen = torch.zeros(n * v, dtype=torch.bool, device="cuda")
    seen[at] = True
    seen = seen.view(n, v)
    count = torch.zeros(n * v, dtype=torch.int32, device="cuda").index_add_(0, at, behind.int()).view(n, v)
    r = p["repetition_penalty"]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = torch.where(count > 0, x - p["frequency_penalty"] * count - p["presence_penalty"], x)
    if s["bias_ids"] is not None:
        total = s["bias_ids"].numel()
        key = _row_of(s["bias_offsets"], total) * v + s["bias_ids"].long()
        last = torch.full((n * v,), -1, dtype=torch.int64, device="cuda")
        last.scatter_reduce_(0, key, torch.arange(total, device="cuda"), "amax")
        last = last.view(n, v)
        x = torch.where(last >= 0, x + s["bias_values"][last.clamp_min(0)], x)
    flags = torch.zeros(n, dtype=torch.int32, device="cuda")
    if s["mask"] is not None:
        bit = torch.arange(32, device="cuda", dtype=torch.int32)
        ok = ((s["mask"][:, :, None] >> bit) & 1).bool().view(s["mask"].shape[0], -1)[:, :v]
        ok = ok[s["mask_rows"].clamp_min(0).long()] | (s["mask_rows"] < 0)[:, None]
        x = torch.where(ok, x, -math.inf)
        flags = torch.where(ok.any(1), 0, EMPTY).int()
    if c["to"] == "inplace":
        s["logits"].copy_(x)
        return dict(logits=s["logits"], flags=flags)
    return dict(logits=x.to(torch.float32 if c["to"] == "f32" else s["logits"].dtype), flags=flags)


# ---- the pass -----------------------------------------------------------------


def run(s):
    c = s["case"]
    if c["kind"] == "rules":
        if not own:
            return _rules(s, c)
        from gemmaedge_amd import rules as R

        flags = torch.empty(c["rows"], dtype=torch.int32, device="cuda")
        out = R.apply(s["logits"], s["config"], out=s["logits"] if c["to"] == "inplace" else None,
                      out_dtype=torch.float32 if c["to"] == "f32" else None, row_params=s["row_params"], history=s["history"],
                      history_offsets=s["offsets"], prompt_len=s["prompt"], bias_ids=s["bias_ids"], bias_values=s["bias_values"],
                      bias_offsets=s["bias_offsets"], mask=s["mask"], mask_rows=s["mask_rows"], flags=flags)
        return dict(logits=out, flags=flags)
    if not own:
        out = dict(out=_project(s, c))
        if c["kind"] == "train":
            out["dh"], out["da"], out["db"] = _project_backward(s, c)
        return out
    adapters = (s["a"], s["b"], s["scale"], s["adapter"])
    out = dict(out=s["projection"].project(s["h"], s["w"], *adapters, out_dtype=DTYPES[c["odtype"]]))
    if c["kind"] == "train":
        out["dh"], out["da"], out["db"] = s["projection"].project_backward(s["dout"], s["h"], s["w"], *adapters)
    return out


def work(case):
    c = case
    size = 2 if c["dtype"] == "bf16" else 4
    n = c["rows"]
    if c["kind"] == "rules":
        v, ids = c["vocab"], n * (c["history"] / 2 + c["bias"])
        to = 4 if c["to"] == "f32" else size
        lists = 4.0 * ids + 4.0 * n * c["bias"] / 2
        masked = 0.0 if c["mask"] == "none" else 6 / 7
        bits = max(1, n // 2) * v / 8.0 if masked else 0.0
        if c["to"] != "inplace" or c["cap"] > 0:
            return dict(bytes=n * v * (size + to) + lists + bits + 4 * n, flops=(20.0 if c["cap"] > 0 else 2.0) * n * v)
        hidden = masked * (1.0 - ALLOWED.get(c["mask"], 1.0))  # logits that are only written
        return dict(bytes=n * v * size * hidden + 2 * size * ids * (1.0 - hidden) + lists + bits + 4 * n, flops=6.0 * ids + 1.0)
    d, v, r = c["dim"], c["out"], c["rank"]
    used = c["adapters"] * (1.0 - (1.0 - 1.0 / c["adapters"]) ** min(n, 40))  # adapters that have rows
    low = used * r * (d + v) * size
    osize = 2 if c["odtype"] == "bf16" else 4
    forward = dict(bytes=(n + v) * d * size + low + n * v * osize + 4 * n, flops=2.0 * n * d * v + 2.0 * n * r * (d + v))
    if c["kind"] == "project":
        return forward
    return dict(bytes=forward["bytes"] + n * (v + d) * size + c["adapters"] * r * (d + v) * size,
                flops=2 * forward["flops"] + 2.0 * n * r * (d + v))


# ---- the definitions in 64 bits -------------------------------------------------


def exact(case, seed):
    c = dict(case)
    s = _inputs(c, seed)
    return _exact_rules(c, s) if c["kind"] == "rules" else _exact_project(c, s)


def _exact_project(c, s):
    n, v, k, r = c["rows"], c["out"], c["adapters"], c["rank"]
    h = s["h"].double()
    a = s["a"].double()
    at = s["adapter"].long()
    # one-hot over adapters, times the scale: rows without an adapter are zeros
    which = torch.zeros(n, k, dtype=torch.float64, device="cuda")
    have = at >= 0
    which[have, at[have]] = s["scale"].double()[at[have]]
    u = (h @ a.view(k * r, -1).t()).view(n, k, r).mul_(which[:, :, None]).view(n, k * r)
    out = torch.empty(n, v, dtype=torch.float64, device="cuda")
    train = c["kind"] == "train"
    dh, du = torch.zeros_like(h), torch.zeros_like(u)
    db = torch.empty(k, v, r, dtype=torch.float64, device="cuda") if train else None
    piece = max(1024, (1 << 28) // max(n, k * r, c["dim"]))  # outputs at a time
    for i in range(0, v, piece):
        j = min(v, i + piece)
        w = s["w"][i:j].double()
        b = s["b"][:, i:j].double().permute(1, 0, 2).reshape(j - i, k * r)
        out[:, i:j] = torch.addmm(h @ w.t(), u, b.t().contiguous())
        if train:
            g = s["dout"][:, i:j].double()
            dh.addmm_(g, w)
            du.addmm_(g, b)
            db[:, i:j] = (g.t() @ u).view(j - i, k, r).permute(1, 0, 2)
    if not train:
        return dict(out=out)
    du = du.view(n, k, r).mul_(which[:, :, None]).view(n, k * r)
    dh.addmm_(du, a.view(k * r, -1))
    return dict(out=out, dh=dh, da=(du.t() @ h).view(k, r, -1), db=db)


def _exact_rules(c, s):
    n, v = c["rows"], c["vocab"]
    cap = c["cap"]
    value = lambda k, i: float(s["params"][k][i, 0]) if c["per_row"] else s["params"][k]  # noqa: E731
    out = torch.empty(n, v, dtype=torch.float64, device="cuda")
    flags = torch.zeros(n, dtype=torch.int32, device="cuda")
    offs, prompt = s["offsets"].tolist(), s["prompt"].tolist()
    bias = s["bias_offsets"].tolist() if s["bias_ids"] is not None else None
    place = torch.arange(v, device="cuda")
    for i in range(n):
        x = s["logits"][i].double()
        if cap > 0:
            e = torch.expm1(2.0 * x / cap)
            x = cap * e / (e + 2.0)
        ids = s["history"][offs[i]:offs[i + 1]].long()
        every, late = torch.bincount(ids, minlength=v), torch.bincount(ids[prompt[i]:], minlength=v)
        r = value("repetition_penalty", i)
        x = torch.where(every > 0, torch.where(x > 0, x / r, x * r), x)
        x -= (late > 0) * value("presence_penalty", i) + late * value("frequency_penalty", i)
        if bias:
            keys, vals = s["bias_ids"][bias[i]:bias[i + 1]].tolist(), s["bias_values"][bias[i]:bias[i + 1]].tolist()
            d = dict(zip(keys, vals))
            if d:
                x[torch.tensor(list(d), device="cuda")] += torch.tensor(list(d.values()), device="cuda", dtype=torch.float64)
        m = int(s["mask_rows"][i]) if s["mask"] is not None else -1
        if m >= 0:
            ok = (s["mask"][m].long()[place // 32] >> (place % 32)) % 2 == 1
            x = x.masked_fill(~ok, -math.inf)
            flags[i] = 0 if bool(ok.any()) else EMPTY
        out[i] = x
    return dict(logits=out, flags=flags)
