"""The operators of one served decode step, as measurable cases.

  step      one new token of each sequence: its key and value into a paged
            cache (int8 codes with a scale a position and head, or float16),
            then attention of its query heads over the sequence's pages, with
            an optional tanh cap of the scores and a bias by distance
  store     prompts' keys and values into the paged cache, and the rows as the
            cache holds them
  quantize  rows into microscaled 4-bit floats (e2m1 codes, one e8m0 scale a
            block of 32), and the values those stand for
  linear    microscaled activations times a microscaled weight matrix, with
            the layers' bias, GELU and residual
  logits    penalties for repeated tokens, biases and a grammar's mask on a
            head's logits, and the greedy pick

Where `own` is false, run() is each operator in plain torch operations; where
it is true, the library's own calls.
"""
import math

import torch

own = False

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------- cases


def listed():
    return [
        # GPT-2's 12 heads of 64 at a prompt's end, one user: latency counts
        {"name": "step gpt2", "kind": "step", "type": "int8", "rows": 1, "heads": 12, "kv": 12, "hd": 64, "page": 64,
         "lo": 477, "hi": 477, "cap": 0.0, "bias": False},
        # a few long documents, grouped heads of 128, the float16 cache, capped scores
        {"name": "step long f16", "kind": "step", "type": "f16", "rows": 4, "heads": 32, "kv": 8, "hd": 128, "page": 256,
         "lo": 9001, "hi": 32768, "cap": 30.0, "bias": False},
        # a full server: 64 ragged conversations, the int8 cache, the distance bias
        {"name": "step batch int8", "kind": "step", "type": "int8", "rows": 64, "heads": 32, "kv": 8, "hd": 128,
         "page": 128, "lo": 130, "hi": 16384, "cap": 0.0, "bias": True},
        # one GPT-2 prompt into its pages
        {"name": "store prompt", "kind": "store", "type": "int8", "rows": 1, "kv": 12, "hd": 64, "page": 64, "lo": 476,
         "hi": 476},
        # eight ragged prompts of a grouped-head model at once
        {"name": "store prompts f16", "kind": "store", "type": "f16", "rows": 8, "kv": 8, "hd": 128, "page": 128,
         "lo": 333, "hi": 4096},
        # 16 sequences' activations before a decode step's matmul
        {"name": "quantize decode", "kind": "quantize", "t": 16, "k": 2048},
        # a prompt's activations between a 7B Llama's gate / up and down
        {"name": "quantize prompt", "kind": "quantize", "t": 4096, "k": 11008},
        # one token through a 7B Llama's gate matrix
        {"name": "linear decode", "kind": "linear", "t": 1, "k": 4096, "n": 11008, "bias": False, "gelu": False,
         "resid": False},
        # a ragged batch of sequences through TinyLlama's down matrix into the residual stream
        {"name": "linear batch", "kind": "linear", "t": 37, "k": 5632, "n": 2048, "bias": True, "gelu": False,
         "resid": True},
        # a long prompt through a 7B Llama's gate matrix
        {"name": "linear prompt", "kind": "linear", "t": 2048, "k": 4096, "n": 11008, "bias": False, "gelu": False,
         "resid": False},
        # one user's next token over TinyLlama's vocabulary
        {"name": "logits one", "kind": "logits", "rows": 1, "v": 32000, "hist": 476, "biases": 16, "mask": True},
        # a full server over GPT-2's vocabulary, long histories
        {"name": "logits batch", "kind": "logits", "rows": 256, "v": 50257, "hist": 2048, "biases": 64, "mask": True},
    ]


def log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("step", "step", "linear", "linear", "store", "quantize", "logits"))
    if kind in ("step", "store"):
        hd = rng.choice((64, 128))
        kv = rng.choice((1, 2, 4, 8, 12))
        c = {"kind": kind, "type": rng.choice(("int8", "f16")), "rows": log_int(rng, 1, 64), "kv": kv, "hd": hd,
             "page": rng.choice((64, 128, 192, 256, 512))}
        most = min(16384 if c["rows"] > 4 else 32768, (1 << (22 if c["type"] == "int8" else 21)) // (c["rows"] * kv))
        if kind == "store":
            most = min(most, max(1, 16384 // c["rows"]))
        c["hi"] = log_int(rng, 1, most)
        c["lo"] = rng.randint(1, c["hi"]) if rng.random() < 0.5 else c["hi"]
        if kind == "step":
            c["heads"] = kv * rng.choice((1, 2, 3, 4, 8))
            c["cap"] = rng.choice((0.0, 0.0, 30.0, 50.0))
            c["bias"] = rng.random() < 0.4
        return c
    if kind == "quantize":
        return {"kind": kind, "t": log_int(rng, 1, 4096), "k": 32 * log_int(rng, 1, 344)}
    if kind == "logits":
        return {"kind": kind, "rows": log_int(rng, 1, 256), "v": log_int(rng, 1000, 50257), "hist": log_int(rng, 1, 2048),
                "biases": rng.choice((0, 3, 64, 300)), "mask": rng.random() < 0.6}
    while True:
        t = 1 if rng.random() < 0.3 else log_int(rng, 2, 2048)
        k = 32 * log_int(rng, 8, 344)
        n = log_int(rng, 200, 12000)
        if t * k * n <= 2048 * 4096 * 11008:
            break
    gelu = rng.random() < 0.3
    return {"kind": kind, "t": t, "k": k, "n": n, "bias": rng.random() < 0.6, "gelu": gelu,
            "resid": not gelu and rng.random() < 0.4}


# ------------------------------------------------------------------ inputs


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 11)
    return g


def normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def activations(g, t, k):
    """Rows of a residual stream: normal, a few channels much larger."""
    x = normal(g, t, k)
    big = torch.randint(0, k, (max(1, k // 256),), generator=g, device="cuda")
    x[:, big] *= 8.0
    return x


def lengths(case):
    """The sequences' lengths in order; their sum is the case's, not the seed's."""
    n = case["rows"]
    return [case["hi"] - (case["hi"] - case["lo"]) * i // max(1, n - 1) for i in range(n)]


def paged(case, seed, g):
    """Lengths in a random order, and a page table over scattered pages."""
    n, page = case["rows"], case["page"]
    order = torch.randperm(n, generator=g, device="cuda")
    length = torch.tensor(lengths(case), dtype=torch.int32, device="cuda")[order]
    need = (length + page - 1) // page
    width = -(-case["hi"] // page)
    n_pages = sum(-(-l // page) for l in lengths(case)) + 3
    free = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    first = torch.cumsum(need, 0) - need
    at = torch.arange(width, device="cuda")[None, :]
    table = torch.where(at < need[:, None], free[(first[:, None] + at).clamp(max=n_pages - 1)], -1).to(torch.int32)
    return length, table.contiguous(), n_pages


def tokens(length):
    """(sequence, position) of every token of the sequences, one after another."""
    n = length.to(torch.int64)
    seq = torch.repeat_interleave(torch.arange(len(n), device="cuda"), n)
    first = torch.cumsum(n, 0) - n
    return seq.to(torch.int32), (torch.arange(len(seq), device="cuda") - first[seq]).to(torch.int32)


def logit_inputs(case, g):
    s, n, v = {}, case["rows"], case["v"]
    s["logits"] = normal(g, n, v, std=3.0)
    count = torch.randint(0, case["hist"] + 1, (n,), generator=g, device="cuda")
    count[0] = case["hist"]
    s["hist_off"] = torch.cat([count.new_zeros(1), torch.cumsum(count, 0)])
    # words come back, the frequent ones most
    u = torch.rand(n * case["hist"], generator=g, device="cuda")
    s["hist"] = (u ** 3 * v).to(torch.int32).clamp(max=v - 1)
    s["rep"] = 1.0 + 0.3 * torch.rand(n, generator=g, device="cuda")
    s["pres"] = 0.5 * torch.rand(n, generator=g, device="cuda")
    s["freq"] = 0.2 * torch.rand(n, generator=g, device="cuda")
    s["bias_off"] = torch.arange(n + 1, device="cuda") * case["biases"]
    s["bias_ids"] = torch.randint(0, v, (n * case["biases"],), generator=g, device="cuda", dtype=torch.int32)
    s["bias"] = normal(g, n * case["biases"], std=4.0)
    s["mask"] = None
    if case["mask"]:  # a grammar's allowed tokens, one bit each
        words = -(-v // 32)
        s["mask"] = torch.randint(-2 ** 31, 2 ** 31, (n, words), generator=g, device="cuda").to(torch.int32)
    return s


def prepare(case, seed):
    g = generator(seed)
    s = {"case": case}
    if own:
        import llm_mojo_amd as lm

        s["lm"], s["ctx"] = lm, lm.Context(0, torch.cuda.current_stream())
    if case["kind"] in ("step", "store"):
        kv, hd, page = case["kv"], case["hd"], case["page"]
        s["length"], s["table"], n_pages = paged(case, seed, g)
        seq, pos = tokens(s["length"])
        s["seq"], s["pos"] = seq, pos
        k = normal(g, len(seq), kv, hd) * (0.25 + normal(g, 1, kv, hd).abs())  # channels of unlike sizes
        v = normal(g, len(seq), kv, hd)
        if case["kind"] == "store":
            s["k"], s["v"] = k, v
        if own:
            s["cache"] = s["lm"].PagedKV(s["ctx"], 1, n_pages, page, kv, hd, case["type"])
        else:  # the cache in its plain form: [page, position in it, head, dimension] and a scale a head's row
            codes = torch.int8 if case["type"] == "int8" else torch.float16
            s["cache"] = [torch.zeros(n_pages, page, kv, hd, dtype=codes, device="cuda") for _ in range(2)]
            s["scale"] = [torch.ones(n_pages, page, kv, device="cuda") for _ in range(2)]
        if case["kind"] == "step":
            n, heads = case["rows"], case["heads"]
            # qkv rows as a fused projection leaves them: query heads, key heads, value heads
            s["qkv"] = normal(g, n, (heads + 2 * kv) * hd)
            s["qkv"][:, :heads * hd] *= 2.0
            s["out"] = torch.zeros(n, heads * hd, device="cuda")
            s["now"] = s["length"] - 1
            s["all"] = torch.arange(n, dtype=torch.int32, device="cuda")
            s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, heads + 1, device="cuda") / heads) if case["bias"] else None
            if own:
                s["cache"].store(0, k, v, seq, pos, s["table"])
                s["work"] = torch.empty(s["cache"].work_bytes(n, heads), dtype=torch.uint8, device="cuda")
                s["ko"], s["vo"] = torch.empty(n, kv, hd, device="cuda"), torch.empty(n, kv, hd, device="cuda")
            else:
                put(s, k, v, seq, pos)
        elif own:
            s["ko"], s["vo"] = torch.empty_like(k), torch.empty_like(v)
    elif case["kind"] == "quantize":
        s["x"] = activations(g, case["t"], case["k"])
        if own:
            t, k = case["t"], case["k"]
            s["codes"] = torch.empty(t, k // 2, dtype=torch.uint8, device="cuda")
            s["scales"] = torch.empty(t, k // 32, dtype=torch.uint8, device="cuda")
            s["values"] = torch.empty(t, k, device="cuda")
    elif case["kind"] == "linear":
        t, k, n = case["t"], case["k"], case["n"]
        s["x"] = activations(g, t, k)
        w = normal(g, n, k, std=0.02)
        s["b"] = normal(g, n, std=0.1) if case["bias"] else None
        s["resid"] = normal(g, t, n) if case["resid"] else None
        s["out"] = torch.zeros(t, n, device="cuda")
        if own:
            s["w"] = s["lm"].HipMX4Matrix.from_f32(s["ctx"], w, reduce_rows=False)
        else:
            s["w"] = pack(*mx4(w))
    else:
        n, v = case["rows"], case["v"]
        s.update(logit_inputs(case, g))
        s["out"] = torch.zeros(n, v, device="cuda")
        s["pick"] = torch.zeros(n, dtype=torch.int64, device="cuda")
        if own:
            s["work"] = torch.empty(s["lm"].logits_work_bytes(n, v), dtype=torch.uint8, device="cuda")
    return s


# --------------------------------------------------------------- plain forms


def rows_of(cache_type, x):
    """Rows as a cache holds them: (codes, scale): round-half-away int8 codes by max|x| / 127 (1 for a zero row), or
    float16 values, saturating."""
    if cache_type == "f16":
        return x.clamp(-65504.0, 65504.0).to(torch.float16), torch.ones_like(x[..., 0])
    sc = x.abs().amax(-1) / 127.0
    sc = torch.where(sc == 0, torch.ones_like(sc), sc)
    y = x * (1.0 / sc)[..., None]
    return (torch.sign(y) * torch.floor(y.abs() + 0.5)).to(torch.int8), sc


def put(s, k, v, seq, pos):
    """Rows into the plain cache."""
    page = s["case"]["page"]
    at = s["table"][seq.long(), pos.long() // page].long()
    (ck, sk), (cv, sv) = rows_of(s["case"]["type"], k), rows_of(s["case"]["type"], v)
    s["cache"][0][at, pos.long() % page], s["scale"][0][at, pos.long() % page] = ck, sk
    s["cache"][1][at, pos.long() % page], s["scale"][1][at, pos.long() % page] = cv, sv


def got(s, seq, pos):
    """Rows of the plain cache as the values they stand for."""
    page = s["case"]["page"]
    at, off = s["table"][seq.long(), pos.long() // page].long(), pos.long() % page
    return tuple(x[at, off].float() * y[at, off][..., None] for x, y in zip(s["cache"], s["scale"]))


def plain_step(s):
    c = s["case"]
    n, heads, kv, hd = c["rows"], c["heads"], c["kv"], c["hd"]
    rows = s["qkv"].view(n, heads + 2 * kv, hd)
    put(s, rows[:, heads:heads + kv], rows[:, heads + kv:], s["all"], s["now"])
    at = s["table"].clamp(min=0).long()  # pages past a sequence's end are masked below

    def dense(i):  # [rows, kv, position, hd]
        x = s["cache"][i][at].float() * s["scale"][i][at][..., None]
        return x.reshape(n, -1, kv, hd).transpose(1, 2).contiguous()

    q = rows[:, :heads].reshape(n, kv, heads // kv, hd)
    k = dense(0)
    score = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(hd)
    if c["cap"]:
        score = c["cap"] * torch.tanh(score / c["cap"])
    j = torch.arange(score.shape[-1], device="cuda")
    if s["slopes"] is not None:
        away = (j[None, :] - s["now"][:, None]).float()
        score = score + s["slopes"].view(1, kv, -1, 1) * away[:, None, None, :]
    seen = (j[None, :] <= s["now"][:, None])[:, None, None, :]
    score = torch.where(seen, score, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    out = torch.matmul(p, dense(1)) / p.sum(-1, keepdim=True)
    return out.reshape(n, heads * hd), *got(s, s["all"], s["now"])


def power(e):
    """2 ** (e - 127) for whole e from 0 to 254."""
    return torch.where(e == 0, torch.full_like(e, 1 << 22), e << 23).view(torch.float32)


def mx4(x):
    """(signed e2m1 values [t, k / 32, 32], scale exponents [t, k / 32]) of finite rows."""
    b = x.reshape(x.shape[0], -1, 32)
    e = ((b.abs().amax(-1).view(torch.int32) >> 23) - 2).clamp(min=0)
    a = (b * power(254 - e)[..., None]).abs()
    # nearest, ties to the even code, at most 6
    i = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    val = torch.tensor(E2M1, device=x.device)[i.to(torch.int32)]
    return torch.where(torch.signbit(b), -val, val), e


def pack(values, e):
    """Two codes a byte (the even column's low) and exponent bytes."""
    a = values.abs()
    i = torch.searchsorted(torch.tensor(E2M1, device=a.device), a.contiguous()).to(torch.uint8)
    i = (i + 8 * torch.signbit(values).to(torch.uint8)).reshape(a.shape[0], -1, 2)
    return i[..., 0] + 16 * i[..., 1], e.to(torch.uint8)


def unpack(codes, e):
    i = torch.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1, 32).to(torch.int32)
    table = torch.tensor(E2M1 + tuple(-x for x in E2M1), device=codes.device)
    return (table[i] * power(e.to(torch.int32))[..., None]).reshape(codes.shape[0], -1)


def scaled(values, e):
    return (values * power(e)[..., None]).reshape(values.shape[0], -1)


def plain_linear(s):
    c = s["case"]
    y = torch.matmul(scaled(*mx4(s["x"])), unpack(*s["w"]).t())
    if s["b"] is not None:
        y = y + s["b"]
    if c["gelu"]:
        y = 0.5 * y * (1.0 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y * y * y)))
    return y if s["resid"] is None else s["resid"] + y


def plain_logits(s):
    n, v = s["logits"].shape
    l = s["logits"]
    at = torch.arange(len(s["hist"]), device="cuda")
    row = torch.bucketize(at, s["hist_off"][1:], right=True)
    live = row < n
    count = torch.zeros(n * v, dtype=torch.int32, device="cuda")
    count.index_add_(0, torch.where(live, row * v + s["hist"], 0), live.to(torch.int32))
    count = count.view(n, v)
    rep = s["rep"][:, None]
    seen = torch.where(l > 0, l / rep, l * rep) - (s["freq"][:, None] * count.float() + s["pres"][:, None])
    l = torch.where(count > 0, seen, l)
    brow = torch.bucketize(torch.arange(len(s["bias"]), device="cuda"), s["bias_off"][1:], right=True)
    add = torch.zeros(n * v, device="cuda").index_add_(0, brow * v + s["bias_ids"], s["bias"])
    l = l + add.view(n, v)
    if s["mask"] is not None:
        i = torch.arange(v, device="cuda")
        l = torch.where((s["mask"][:, i >> 5] >> (i & 31)) & 1 != 0, l, -math.inf)
    best = l.amax(-1)
    return {"logits": l, "pick": torch.where(best > -math.inf, torch.argmax(l, -1), -1)}


# --------------------------------------------------------------------- run


def run(s):
    c = s["case"]
    if c["kind"] == "step":
        if own:
            n, heads, kv, hd = c["rows"], c["heads"], c["kv"], c["hd"]
            rows = s["qkv"].view(n, heads + 2 * kv, hd)
            s["cache"].step(0, s["out"], rows[:, :heads], rows[:, heads:heads + kv], rows[:, heads + kv:], s["now"],
                            s["table"], s["work"], cap=c["cap"], slopes=s["slopes"])
            s["cache"].fetch(0, s["ko"], s["vo"], s["all"], s["now"], s["table"])  # what the step left there
            return s["out"], s["ko"], s["vo"]
        return plain_step(s)
    if c["kind"] == "store":
        if own:
            s["cache"].store(0, s["k"], s["v"], s["seq"], s["pos"], s["table"])
            s["cache"].fetch(0, s["ko"], s["vo"], s["seq"], s["pos"], s["table"])
            return s["ko"], s["vo"]
        put(s, s["k"], s["v"], s["seq"], s["pos"])
        return got(s, s["seq"], s["pos"])
    if c["kind"] == "quantize":
        if own:
            s["lm"].mx4_quantize(s["ctx"], s["x"], s["codes"], s["scales"])
            s["lm"].mx4_dequantize(s["ctx"], s["codes"], s["scales"], s["values"])
            return s["values"]
        return scaled(*mx4(s["x"]))
    if c["kind"] == "linear":
        if own:
            if c["resid"]:
                s["out"].copy_(s["resid"])
            s["lm"].linear(s["ctx"], s["out"], s["x"], s["w"], s["b"], resid=c["resid"], gelu=c["gelu"])
            return s["out"]
        return plain_linear(s)
    if own:
        s["lm"].adjust_logits(s["ctx"], s["out"], s["logits"], history=(s["hist"], s["hist_off"]), repetition=s["rep"],
                              presence=s["pres"], frequency=s["freq"], bias=(s["bias_ids"], s["bias"], s["bias_off"]),
                              mask=s["mask"], pick=s["pick"], work=s["work"])
        return {"logits": s["out"], "pick": s["pick"]}
    return plain_logits(s)


def work(case):
    c = case
    if c["kind"] == "step":
        n, per = sum(lengths(c)), c["hd"] * (1 if c["type"] == "int8" else 2) + (4 if c["type"] == "int8" else 0)
        return {"bytes": 2 * n * c["kv"] * per + 4 * c["rows"] * c["hd"] * 2 * (c["heads"] + 2 * c["kv"]),
                "flops": 4 * n * c["heads"] * c["hd"]}
    if c["kind"] == "store":  # rows in, the cache written and read, rows out
        n, per = sum(lengths(c)), c["hd"] * (1 if c["type"] == "int8" else 2) + (4 if c["type"] == "int8" else 0)
        return {"bytes": 2 * n * c["kv"] * (8 * c["hd"] + 2 * per), "flops": 0}
    if c["kind"] == "quantize":  # rows in, codes and scales written and read, values out
        return {"bytes": c["t"] * c["k"] * (8 + 2 * 17 / 32), "flops": 0}
    if c["kind"] == "linear":
        t, k, n = c["t"], c["k"], c["n"]
        return {"bytes": n * k * 17 / 32 + 4 * t * k + 4 * t * n * (3 if c["resid"] else 1) + (4 * n if c["bias"] else 0),
                "flops": 2 * t * k * n}
    n, v = c["rows"], c["v"]
    return {"bytes": n * (8 * v + (v / 8 if c["mask"] else 0) + 4 * c["hist"] / 2 + 8 * c["biases"] + 32), "flops": 0}


# ------------------------------------------------------- the definitions in 64 bits


def exact_values(x):
    """A row's microscaled values: 2 ** floor(log2 max|x|) / 4 times the nearest of E2M1, ties to the even code."""
    b = x.double().reshape(x.shape[0], -1, 32)
    _, e = torch.frexp(b.abs().amax(-1, keepdim=True))
    unit = torch.ldexp(torch.ones_like(e, dtype=torch.float64), (e - 3).clamp(min=-127))
    grid = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    mid = (grid[1:] + grid[:-1]) / 2
    a = b.abs() / unit
    low = torch.bucketize(a, mid)  # a tie: the code below it
    high = torch.bucketize(a, mid, right=True)
    return (torch.sign(b) * grid[torch.where(low % 2 == 0, low, high)] * unit).reshape(x.shape)


def exact_row(kind, x):
    """Rows as the cache's values."""
    if kind == "f16":
        return x.clamp(-65504.0, 65504.0).half().double()
    size = x.abs().amax(-1, keepdim=True)
    sc = torch.where(size == 0, torch.ones_like(size), size / 127.0)
    y = x * (1.0 / sc)
    return torch.where(y < 0, torch.ceil(y.double() - 0.5), torch.floor(y.double() + 0.5)) * sc.double()


def exact(case, seed):
    c = dict(case)
    g = generator(seed)
    if c["kind"] in ("step", "store"):
        length, table, _ = paged(c, seed, g)
        seq, pos = tokens(length)
        k = normal(g, len(seq), c["kv"], c["hd"]) * (0.25 + normal(g, 1, c["kv"], c["hd"]).abs())
        v = normal(g, len(seq), c["kv"], c["hd"])
        if c["kind"] == "store":
            return exact_row(c["type"], k), exact_row(c["type"], v)
        n, h, kv, hd = c["rows"], c["heads"], c["kv"], c["hd"]
        qkv = normal(g, n, (h + 2 * kv) * hd)
        qkv[:, :h * hd] *= 2.0
        qkv = qkv.view(n, h + 2 * kv, hd)
        out = torch.zeros(n, h, hd, dtype=torch.float64, device="cuda")
        new = [torch.zeros(n, kv, hd, dtype=torch.float64, device="cuda") for _ in range(2)]
        first = 0
        for r in range(n):
            m = int(length[r])
            kr, vr = k[first:first + m].clone(), v[first:first + m].clone()
            first += m
            kr[-1], vr[-1] = qkv[r, h:h + kv], qkv[r, h + kv:]
            kr, vr = exact_row(c["type"], kr), exact_row(c["type"], vr)
            new[0][r], new[1][r] = kr[-1], vr[-1]
            q = qkv[r, :h].double().view(kv, h // kv, hd)
            sc = torch.matmul(q, kr.permute(1, 2, 0).contiguous()) * hd ** -0.5
            if c["cap"]:
                sc = torch.tanh(sc / c["cap"]) * c["cap"]
            if c["bias"]:
                # the slopes are inputs, in 32 bits
                sl = (2.0 ** (-8.0 * torch.arange(1, h + 1, device="cuda") / h)).double().view(kv, h // kv, 1)
                sc = sc - sl * torch.arange(m - 1, -1, -1, device="cuda")
            p = torch.softmax(sc, -1)
            out[r] = torch.matmul(p, vr.permute(1, 0, 2).contiguous()).reshape(h, hd)
        return out.reshape(n, h * hd), *new
    if c["kind"] == "quantize":
        return exact_values(activations(g, c["t"], c["k"]))
    if c["kind"] == "linear":
        x = activations(g, c["t"], c["k"])
        w = normal(g, c["n"], c["k"], std=0.02)
        b = normal(g, c["n"], std=0.1) if c["bias"] else None
        y = torch.matmul(exact_values(x), exact_values(w).t())
        if b is not None:
            y = y + b
        if c["gelu"]:
            y = y / 2 * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
        return normal(g, c["t"], c["n"]).double() + y if c["resid"] else y
    s = logit_inputs(c, g)
    n, v = c["rows"], c["v"]
    l = s["logits"].double()
    off, boff = s["hist_off"].tolist(), s["bias_off"].tolist()
    for r in range(n):
        count = torch.bincount(s["hist"][off[r]:off[r + 1]].long(), minlength=v)
        hit, rep = count > 0, float(s["rep"][r])
        y = l[r]
        y = torch.where(hit & (y > 0), y / rep, torch.where(hit, y * rep, y))
        y = y - hit * (float(s["freq"][r]) * count + float(s["pres"][r]))
        ids = s["bias_ids"][boff[r]:boff[r + 1]].long()
        y = y.scatter_add(0, ids, s["bias"][boff[r]:boff[r + 1]].double())
        if s["mask"] is not None:
            shifts = torch.arange(32, device="cuda", dtype=torch.int32)
            bit = ((s["mask"][r][:, None] >> shifts) & 1).reshape(-1)[:v]
            y = y.masked_fill(bit == 0, -math.inf)
        l[r] = y
    return {"logits": l, "pick": None}
