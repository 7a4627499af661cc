"""The serving operators over a paged key-value cache, and the rules on logits, as measured cases.

append           new tokens' key and value rows into the pages of a cache
attend           attention of one new token per sequence over its pages, with a sliding window and
                 first tokens that stay visible (sinks), and with the accumulated attention weights
attend_prompt    the same attention for the tokens of a prompt (or a chunk of one)
evict            a cache cut down to a budget of slots per key-value head by accumulated weight
adjust_logits    penalties for repeated tokens, biases, a grammar mask, and the greedy pick

Where `own` is false `run` computes the plain form with elementary torch operations.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ESIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one decode step's new rows of 64 conversations (Qwen3-0.6B's 8 kv heads of 128), from the fp32 rows of a decode
        # engine; the cache keeps the attention weights
        dict(name="append_step_b64", op="append", batch=64, new=1, ragged=False, cached=700, n_kv=8, head_dim=128, page=16,
             dtype="bf16", src="fp32", track=True),
        # the rows of four prompts of up to 2048 tokens behind nothing, one wide kv head (Gemma 3 1B)
        dict(name="append_prompts_b4", op="append", batch=4, new=2048, ragged=True, cached=0, n_kv=1, head_dim=256, page=64,
             dtype="fp16", src="fp16", track=False),
        # one conversation on a sliding layer (Gemma 3 1B: 4 heads on 1, window 512): latency counts
        dict(name="attend_window_b1", op="attend", batch=1, length=1533, ragged=False, n_heads=4, n_kv=1, head_dim=256,
             page=16, dtype="bf16", window=512, sinks=4, track=False),
        # a full server batch of ragged conversations (Qwen3-0.6B: 16 heads on 8)
        dict(name="attend_b64", op="attend", batch=64, length=8192, ragged=True, n_heads=16, n_kv=8, head_dim=128,
             page=16, dtype="bf16", window=0, sinks=0, track=False),
        # a few long conversations whose attention weights are accumulated for eviction (Qwen3.5: 8 heads on 2 of 256)
        dict(name="attend_weights_b3_long", op="attend", batch=3, length=50001, ragged=True, n_heads=8, n_kv=2, head_dim=256,
             page=64, dtype="fp16", window=0, sinks=0, track=True),
        # chunks of 4 tokens of 8 conversations behind about a thousand cached ones (the engine's prompt chunk)
        dict(name="prompt_chunk4_b8", op="prompt", batch=8, new=4, cached=1001, ragged=True, n_heads=16, n_kv=8, head_dim=128,
             page=16, dtype="bf16", window=0, sinks=0),
        # three whole prompts of up to 8192 tokens, all earlier tokens visible
        dict(name="prompt_full_b3", op="prompt", batch=3, new=8192, cached=0, ragged=True, n_heads=16, n_kv=8, head_dim=128,
             page=64, dtype="bf16", window=0, sinks=0),
        # one long prompt on a sliding layer with sinks (Gemma 3 1B), behind an odd number of cached tokens
        dict(name="prompt_window_b1", op="prompt", batch=1, new=16000, cached=777, ragged=False, n_heads=4, n_kv=1,
             head_dim=256, page=16, dtype="fp16", window=512, sinks=4),
        # the steady state: every conversation one token over its budget
        dict(name="evict_step_b16", op="evict", batch=16, length=1025, ragged=False, budget=1024, sinks=4, recent=256, n_kv=8,
             head_dim=128, page=16, dtype="bf16"),
        # long ragged conversations cut to a quarter, some of them below the budget
        dict(name="evict_long_b6", op="evict", batch=6, length=8192, ragged=True, budget=2048, sinks=4, recent=512, n_kv=8,
             head_dim=128, page=64, dtype="bf16"),
        # one conversation (Qwen3's vocabulary) with a grammar mask
        dict(name="logits_b1", op="logits", rows=1, vocab=151936, history=500, biases=20, mask=True),
        # a server batch (Gemma 3's vocabulary), long histories and biases
        dict(name="logits_b64", op="logits", rows=64, vocab=262144, history=4000, biases=300, mask=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "prompt", "prompt", "evict", "logits"])
    heads = dict(n_kv=rng.choice([1, 2, 4, 8]), head_dim=rng.choice([64, 128, 256]), page=rng.choice([16, 32, 64, 128]),
                 dtype=rng.choice(["bf16", "fp16"]))
    width = heads["n_kv"] * heads["head_dim"]
    group = rng.choice([1, 2, 3, 4, 7, 8])
    masks = dict(window=rng.choice([0, 0, _log(rng, 1, 4096)]), sinks=rng.choice([0, 1, 4, rng.randint(1, 200)]))
    if op == "append":
        batch, new = _log(rng, 1, 64), _log(rng, 1, 2048)
        new = max(1, min(new, (8 << 20) // (batch * width)))
        return dict(op=op, batch=batch, new=new, ragged=rng.random() < 0.5, cached=rng.choice([0, rng.randint(1, 700)]),
                    src=rng.choice(["fp32", heads["dtype"]]), track=rng.random() < 0.5, **heads)
    if op == "attend":
        batch, length = _log(rng, 1, 96), _log(rng, 1, 100000)
        length = max(1, min(length, (1 << 28) // (batch * width)))
        return dict(op=op, batch=batch, length=length, ragged=rng.random() < 0.7, n_heads=heads["n_kv"] * group,
                    track=rng.random() < 0.3, **masks, **heads)
    if op == "prompt":
        batch, new = _log(rng, 1, 16), _log(rng, 1, 8192)
        cached = rng.choice([0, _log(rng, 1, 4096)])
        cost = batch * new * (new + cached) * width * group
        while cost > 8192 * 8192 * 2048:
            new, cached = new // 2 + 1, cached // 2
            batch = batch // 2 + 1
            cost = batch * new * (new + cached) * width * group
        return dict(op=op, batch=batch, new=new, cached=cached, ragged=rng.random() < 0.6, n_heads=heads["n_kv"] * group,
                    **masks, **heads)
    if op == "evict":
        batch, length = _log(rng, 1, 32), _log(rng, 2, 20000)
        length = max(2, min(length, (48 << 20) // (batch * width)))
        budget = rng.randint(max(1, length // 8), length)
        sinks = rng.randint(0, min(8, budget))
        return dict(op=op, batch=batch, length=length, ragged=rng.random() < 0.6, budget=budget, sinks=sinks,
                    recent=rng.randint(0, (budget - sinks) // 2), **heads)
    return dict(op=op, rows=_log(rng, 1, 96), vocab=_log(rng, 100, 170000), history=_log(rng, 1, 8000),
                biases=rng.choice([0, rng.randint(1, 300)]), mask=rng.random() < 0.6)


# -------------------------------------------------------------------------------------- prepare
def _lengths(case, top):
    """Each sequence's token count: `top`, or ragged ones spread evenly over 1 .. top whose first is top."""
    n = case["batch"]
    if not case["ragged"]:
        return [top] * n
    return [top] + [1 + int((b * 0.6180339887498949) % 1 * (top - 1)) for b in range(1, n)]


def _cache(case, lens, g):
    """The pools, the shuffled page lists and the lengths of a cache of these sequences."""
    ps, kv, hd, T = case["page"], case["n_kv"], case["head_dim"], DTYPES[case["dtype"]]
    width = max(-(-n // ps) for n in lens)
    width = max(1, width)
    need = [-(-n // ps) for n in lens]
    total = sum(need) + 2
    perm = torch.randperm(total, device="cuda", generator=g, dtype=torch.int64).to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    # pages of [kv head][slot][head dim], seen as [slot][kv head][head dim]
    k = torch.randn(total, kv, ps, hd, device="cuda", generator=g, dtype=torch.float32).to(T).permute(0, 2, 1, 3)
    v = torch.randn(total, kv, ps, hd, device="cuda", generator=g, dtype=torch.float32).to(T).permute(0, 2, 1, 3)
    length = torch.tensor(lens, dtype=torch.int32, device="cuda")
    return dict(k=k, v=v, table=table, length=length, cap=width * ps)


def _handle(st):
    if own:
        from opentars_b200 import serving
        st["cache"] = serving.PagedCache(st["k"], st["v"], st["table"], st["length"], weight=st.get("weight"),
                                         pos=st.get("pos"), seen=st.get("seen"))
    return st


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.Generator().manual_seed(seed)
    op = case["op"]
    st = dict(case=case)
    if op == "logits":
        R, V, H = case["rows"], case["vocab"], case["history"]
        st["logits"] = torch.randn(R, V, device="cuda", generator=g) * 3
        st["out"] = torch.empty_like(st["logits"])
        # frequent words repeat: squared uniforms crowd the low token ids
        st["history"] = (torch.rand(R, H, device="cuda", generator=g) ** 2 * V).to(torch.int32).clamp_(0, V - 1)
        n_hist = torch.randint(0, H + 1, (R,), generator=h)
        n_hist[0] = H
        st["n_history"] = n_hist.to(torch.int32).cuda()
        st["n_prompt"] = (n_hist // 3).to(torch.int32).cuda()
        st["repetition"] = 1 + torch.rand(R, device="cuda", generator=g)
        st["presence"] = torch.rand(R, device="cuda", generator=g)
        st["frequency"] = torch.rand(R, device="cuda", generator=g) * 0.5
        st["bias_ids"] = st["bias"] = st["mask"] = None
        if case["biases"]:
            st["bias_ids"] = torch.randint(0, V, (R, case["biases"]), device="cuda", generator=g, dtype=torch.int32)
            st["bias"] = torch.randn(R, case["biases"], device="cuda", generator=g) * 5
        if case["mask"]:
            words = -(-V // 32)
            st["mask"] = torch.randint(-(1 << 31), 1 << 31, (R, words), device="cuda", generator=g).to(torch.int32)
        return st
    if op in ("append", "prompt"):
        new = _lengths(case, case["new"])
        lens = [case["cached"] + n for n in new]
        st["new"], st["lens"] = new, lens
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        st["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
    else:
        lens = _lengths(case, case["length"])
        st["lens"] = lens
    st.update(_cache(case, lens, g))
    B, kv, hd, cap, T = len(lens), case["n_kv"], case["head_dim"], st["cap"], DTYPES[case["dtype"]]
    if op == "append":
        src = DTYPES[case["src"]]
        st["k_new"] = torch.randn(cu[-1], kv, hd, device="cuda", generator=g).to(src)
        st["v_new"] = torch.randn(cu[-1], kv, hd, device="cuda", generator=g).to(src)
    if op in ("attend", "prompt"):
        rows = B if op == "attend" else cu[-1]
        st["q"] = (torch.randn(rows, case["n_heads"], hd, device="cuda", generator=g) * 1.5).to(T)
        st["out"] = torch.empty_like(st["q"])
        st["scale"] = hd ** -0.5
    if op == "evict" or case.get("track"):
        # most tokens draw little attention, a few much; some none at all
        w = torch.exp(2 * torch.randn(B, kv, cap, device="cuda", generator=g))
        st["weight"] = torch.where(torch.rand(B, kv, cap, device="cuda", generator=g) < 0.05, torch.zeros_like(w), w)
        st["pos"] = torch.arange(cap, dtype=torch.int32, device="cuda").repeat(B, kv, 1)
        st["seen"] = st["length"].clone()
        st["weight_out"] = torch.zeros_like(w)
    if op == "evict":
        st["pos_out"] = torch.zeros_like(st["pos"])
        st["length_out"] = torch.zeros_like(st["length"])
    return _handle(st)


# ------------------------------------------------------------------------------- the plain forms
def _rows(st, b, n):
    """Where the first n slots of sequence b are: their pages and the rows in them."""
    ps = st["case"]["page"]
    s = torch.arange(n, device="cuda")
    return st["table"][b].long()[s // ps], s % ps


def _plain_append(st):
    T = st["k"].dtype
    at = 0
    for b, (n, total) in enumerate(zip(st["new"], st["lens"])):
        page, row = _rows(st, b, total)
        st["k"][page[total - n:], row[total - n:]] = st["k_new"][at:at + n].to(T)
        st["v"][page[total - n:], row[total - n:]] = st["v_new"][at:at + n].to(T)
        if "weight" in st:
            st["weight"][b, :, total - n:total] = 0
            st["pos"][b, :, total - n:total] = torch.arange(total - n, total, dtype=torch.int32, device="cuda")
        at += n
    return _kept(st)


def _kept(st):
    out = dict(k=st["k"], v=st["v"])
    if "weight" in st:
        out.update(weight=st["weight"], pos=st["pos"])
    return out


def _plain_attend(st):
    c = st["case"]
    G = c["n_heads"] // c["n_kv"]
    if "weight" in st:
        st["weight_out"].copy_(st["weight"])
    for b, n in enumerate(st["lens"]):
        page, row = _rows(st, b, n)
        k = st["k"][page, row].float().permute(1, 2, 0)                  # [kv, hd, n]
        v = st["v"][page, row].float().permute(1, 0, 2)                  # [kv, n, hd]
        q = st["q"][b].float().reshape(c["n_kv"], G, -1) * st["scale"]
        s = q @ k
        if c["window"]:
            j = torch.arange(n, device="cuda")
            s = torch.where((j >= n - c["window"]) | (j < c["sinks"]), s, torch.full_like(s, -math.inf))
        p = torch.exp(s - s.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        st["out"][b] = (p @ v).reshape(c["n_heads"], -1).to(st["q"].dtype)
        if "weight" in st:
            st["weight_out"][b, :, :n] += p.sum(1)
    return dict(out=st["out"], weight=st["weight_out"]) if "weight" in st else st["out"]


def _visible(c, new, total):
    p = torch.arange(total - new, total, device="cuda")[:, None]
    j = torch.arange(total, device="cuda")[None]
    see = j <= p
    return see & ((p - j < c["window"]) | (j < c["sinks"])) if c["window"] else see


def _plain_prompt(st):
    c = st["case"]
    G, at = c["n_heads"] // c["n_kv"], 0
    for b, (new, total) in enumerate(zip(st["new"], st["lens"])):
        page, row = _rows(st, b, total)
        hide = ~_visible(c, new, total)
        for h in range(c["n_kv"]):
            k, v = st["k"][page, row, h].float(), st["v"][page, row, h].float()
            for i in range(h * G, h * G + G):
                s = (st["q"][at:at + new, i].float() * st["scale"]) @ k.T
                s.masked_fill_(hide, -math.inf)
                s = torch.exp_(s.sub_(s.amax(-1, keepdim=True)))
                st["out"][at:at + new, i] = ((s @ v) / s.sum(-1, keepdim=True)).to(st["q"].dtype)
        at += new
    return st["out"]


def _plain_evict(st):
    c = st["case"]
    budget = c["budget"]
    for b, n in enumerate(st["lens"]):
        kept = min(n, budget)
        st["length_out"][b] = kept
        st["weight_out"][b, :, :kept] = st["weight"][b, :, :kept]
        st["pos_out"][b, :, :kept] = st["pos"][b, :, :kept]
        if n <= budget:
            continue
        w, pos = st["weight"][b, :, :n], st["pos"][b, :, :n]
        must = (pos < c["sinks"]) | (pos >= st["seen"][b] - c["recent"])
        order = torch.argsort(torch.where(must, torch.full_like(w, math.inf), w), dim=-1, descending=True, stable=True)
        keep = torch.zeros_like(must).scatter_(1, order[:, :budget], True)
        # as many kept slots lie behind the budget as evicted ones before it; the lists behind that count
        # name kept slots before the budget, which are written onto themselves
        most = min(budget, n - budget)
        dst = torch.argsort(keep[:, :budget].int(), dim=-1, stable=True)[:, :most]
        src = torch.argsort((~keep[:, budget:]).int(), dim=-1, stable=True)[:, :most] + budget
        live = torch.arange(most, device="cuda") < keep[:, budget:].sum(-1, keepdim=True)
        src = torch.where(live, src, dst)
        page, row = _rows(st, b, n)
        head = torch.arange(c["n_kv"], device="cuda")[:, None]
        for pool in (st["k"], st["v"]):
            pool[page[dst], row[dst], head] = pool[page[src], row[src], head]
        st["weight_out"][b, head, dst] = w.gather(1, src)
        st["pos_out"][b, head, dst] = pos.gather(1, src)
    return dict(k=st["k"], v=st["v"], length=st["length_out"], weight=st["weight_out"], pos=st["pos_out"])


def _plain_logits(st):
    x, hist = st["logits"], st["history"].long()
    R, V = x.shape
    at = torch.arange(hist.shape[1], device="cuda")[None]
    there = at < st["n_history"][:, None]
    made = there & (at >= st["n_prompt"][:, None])
    seen = torch.zeros(R, V, device="cuda").scatter_add_(1, hist, there.float()) > 0
    count = torch.zeros(R, V, device="cuda").scatter_add_(1, hist, made.float())
    rep = st["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - st["frequency"][:, None] * count
    x = torch.where(count > 0, x - st["presence"][:, None], x)
    if st["bias"] is not None:
        n = st["bias"].shape[1]
        which = torch.zeros(R, V, dtype=torch.int64, device="cuda")
        which.scatter_reduce_(1, st["bias_ids"].long(), torch.arange(1, n + 1, device="cuda").expand(R, n), "amax")
        x = torch.where(which > 0, x + st["bias"].gather(1, (which - 1).clamp_(min=0)), x)
    if st["mask"] is not None:
        t = torch.arange(V, device="cuda")
        bits = st["mask"][:, t // 32] >> (t % 32).to(torch.int32) & 1
        x = torch.where(bits == 1, x, torch.full_like(x, -math.inf))
    top = torch.where(x == x.amax(-1, keepdim=True), torch.arange(V, device="cuda"), V).amin(-1)
    return dict(logits=x, token=top.to(torch.int32))


PLAIN = dict(append=_plain_append, attend=_plain_attend, prompt=_plain_prompt, evict=_plain_evict, logits=_plain_logits)


# ------------------------------------------------------------------------------- a user's calls
def _own(st):
    from opentars_b200 import serving as S
    c = st["case"]
    op = c["op"]
    if op == "logits":
        token = S.adjust_logits(st["logits"], history=st["history"], n_history=st["n_history"], n_prompt=st["n_prompt"],
                                repetition=st["repetition"], presence=st["presence"], frequency=st["frequency"],
                                bias_ids=st["bias_ids"], bias=st["bias"], mask=st["mask"], out=st["out"])
        return dict(logits=st["out"], token=token)
    cache = st["cache"]
    if op == "append":
        S.append(cache, st["k_new"], st["v_new"], st["cu"])
        return _kept(st)
    if op == "attend":
        if "weight" in st:
            st["weight_out"].copy_(st["weight"])            # the call writes the slots in use only
        out = S.attend(cache, st["q"], st["scale"], window=c["window"], sinks=c["sinks"], out=st["out"],
                       weight_out=st.get("weight_out"))
        return dict(out=out, weight=st["weight_out"]) if "weight" in st else out
    if op == "prompt":
        return S.attend_prompt(cache, st["q"], st["cu"], st["scale"], window=c["window"], sinks=c["sinks"], out=st["out"])
    S.evict(cache, c["budget"], sinks=c["sinks"], recent=c["recent"], length_out=st["length_out"],
            weight_out=st["weight_out"], pos_out=st["pos_out"])
    return dict(k=st["k"], v=st["v"], length=st["length_out"], weight=st["weight_out"], pos=st["pos_out"])


def run(state):
    return _own(state) if own else PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------- the work
def work(case):
    op = case["op"]
    if op == "logits":
        R, V = case["rows"], case["vocab"]
        nbytes = R * (8 * V + (4 * -(-V // 32) if case["mask"] else 0) + 4 * case["history"] // 2 + 8 * case["biases"])
        return dict(bytes=nbytes, flops=3 * R * V)
    kv, hd, e = case["n_kv"], case["head_dim"], 2
    mean = lambda top: top * (0.5 + 0.5 / case["batch"]) if case["ragged"] else top  # noqa: E731
    if op == "append":
        rows = case["batch"] * mean(case["new"])
        return dict(bytes=int(rows * kv * (2 * hd * (ESIZE[case["src"]] + e) + (8 if case["track"] else 0))), flops=0)
    if op == "evict":
        slots = case["batch"] * mean(case["length"]) * kv
        gone = max(0.0, mean(case["length"]) - case["budget"]) * case["batch"] * kv
        kept = min(mean(case["length"]), case["budget"]) * case["batch"] * kv
        moved = gone * kept / max(slots, 1)
        return dict(bytes=int(slots * 8 + kept * 8 + moved * 4 * hd * e), flops=0)
    nh = case["n_heads"]
    if op == "attend":
        n = mean(case["length"])
        see = min(n, case["window"] + case["sinks"]) if case["window"] else n
        nbytes = case["batch"] * (2 * see * kv * hd * e + 2 * nh * hd * e + (8 * n * kv if case["track"] else 0))
        return dict(bytes=int(nbytes), flops=int(4 * case["batch"] * see * nh * hd))
    new = mean(case["new"])
    total = new + case["cached"]
    pairs = new * case["cached"] + new * new / 2
    if case["window"]:
        pairs = min(pairs, new * (case["window"] + case["sinks"]))
    rows = case["batch"] * new
    nbytes = case["batch"] * 2 * min(total, new + case["window"] + case["sinks"] if case["window"] else total) * kv * hd * e
    return dict(bytes=int(nbytes + 2 * rows * nh * hd * e), flops=int(4 * case["batch"] * pairs * nh * hd))


# ------------------------------------------------------------------------- the definitions in 64 bits
def _slots(st, b, n, pool):
    """The first n slots of sequence b, gathered page by page: [n, kv head, head dim] in 64 bits."""
    pages = st["table"][b, :-(-n // st["case"]["page"])].tolist()
    return torch.cat([pool[p] for p in pages])[:n].double()


def _exact_attention(st, b, q, first, total, window, sinks):
    """Rows q [rows, heads, hd] whose first has position `first`: outputs and weights [rows, heads, total]."""
    kv = st["case"]["n_kv"]
    k, v = _slots(st, b, total, st["k"]), _slots(st, b, total, st["v"])
    out = torch.empty_like(q, dtype=torch.float64)
    sums = torch.zeros(kv, total, dtype=torch.float64, device="cuda")
    j = torch.arange(total, device="cuda")
    group = q.shape[1] // kv
    for lo in range(0, q.shape[0], 2048):
        part = q[lo:lo + 2048].double()
        p = torch.arange(first + lo, first + lo + part.shape[0], device="cuda")
        away = p[:, None] - j[None]
        see = (away >= 0) if not window else (away >= 0) & ((away < window) | (j[None] < sinks))
        for i in range(q.shape[1]):
            s = torch.einsum("rd,nd->rn", part[:, i], k[:, i // group]) * st["scale"]
            s = torch.softmax(s.masked_fill(~see, -math.inf), dim=-1)
            out[lo:lo + part.shape[0], i] = torch.einsum("rn,nd->rd", s, v[:, i // group])
            if part.shape[0] == 1:
                sums[i // group] += s[0]
    return out, sums


def _exact_evict(st):
    c = st["case"]
    k, v = st["k"].double(), st["v"].double()
    weight, pos, length = st["weight_out"].double(), st["pos_out"].clone(), st["length_out"].clone()
    ps = c["page"]
    table = st["table"].tolist()
    for b, n in enumerate(st["lens"]):
        length[b] = min(n, c["budget"])
        for h in range(c["n_kv"]):
            w, p = st["weight"][b, h, :n].cpu().numpy().astype("float64"), st["pos"][b, h, :n].cpu().numpy()
            kept = min(n, c["budget"])
            w_new, p_new = w[:kept].copy(), p[:kept].copy()
            if n > kept:
                must = (p < c["sinks"]) | (p >= n - c["recent"])
                ranked = sorted(range(n), key=lambda s: (not must[s], 0.0 if must[s] else -w[s], s))
                stay = set(ranked[:kept])
                holes = [s for s in range(kept) if s not in stay]
                for dst, src in zip(holes, sorted(s for s in stay if s >= kept)):
                    w_new[dst], p_new[dst] = w[src], p[src]
                src = [s for s in sorted(stay) if s >= kept]
                at = lambda ss: ([table[b][s // ps] for s in ss], [s % ps for s in ss])  # noqa: E731
                (sp, sr), (dp, dr) = at(src), at(holes)
                k[dp, dr, h] = st["k"][sp, sr, h].double()
                v[dp, dr, h] = st["v"][sp, sr, h].double()
            weight[b, h, :kept] = torch.from_numpy(w_new).cuda()
            pos[b, h, :kept] = torch.from_numpy(p_new).cuda()
    return dict(k=k, v=v, length=length, weight=weight, pos=pos)


def _exact_logits(st):
    hist, n_all, n_first = (st[k].cpu() for k in ("history", "n_history", "n_prompt"))
    x = st["logits"].double().clone()
    for r in range(x.shape[0]):
        a, f = int(n_all[r]), int(n_first[r])
        ids = torch.unique(hist[r, :a]).long().cuda()
        rep = st["repetition"][r].double()
        x[r, ids] = torch.where(x[r, ids] > 0, x[r, ids] / rep, x[r, ids] * rep)
        ids, count = torch.unique(hist[r, f:a], return_counts=True)
        ids = ids.long().cuda()
        x[r, ids] -= st["frequency"][r].double() * count.cuda().double() + st["presence"][r].double()
        if st["bias"] is not None:
            last = {int(t): float(v) for t, v in zip(st["bias_ids"][r].cpu(), st["bias"][r].cpu())}
            x[r, list(last)] += torch.tensor(list(last.values()), dtype=torch.float64, device="cuda")
        if st["mask"] is not None:
            words = st["mask"][r].cpu().numpy().view("uint32")
            allowed = ((words[:, None] >> torch.arange(32).numpy().astype("uint32")) & 1).reshape(-1)[:x.shape[1]]
            x[r].masked_fill_(torch.from_numpy(allowed == 0).cuda(), -math.inf)
    return dict(logits=x, token=None)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    op = case["op"]
    if op == "logits":
        return _exact_logits(st)
    if op == "evict":
        return _exact_evict(st) if sum(st["lens"]) * case["n_kv"] < 4e6 else None
    if op == "append":
        out = dict(k=st["k"].double(), v=st["v"].double())
        at = 0
        for b, (new, total) in enumerate(zip(st["new"], st["lens"])):
            for i in range(new):
                slot = total - new + i
                page = st["table"][b, slot // case["page"]]
                out["k"][page, slot % case["page"]] = st["k_new"][at + i].double()
                out["v"][page, slot % case["page"]] = st["v_new"][at + i].double()
            at += new
        if "weight" in st:
            weight, pos = st["weight"].double(), st["pos"].clone()
            for b, (new, total) in enumerate(zip(st["new"], st["lens"])):
                weight[b, :, total - new:total] = 0
                pos[b, :, total - new:total] = torch.arange(total - new, total, device="cuda").int()
            out.update(weight=weight, pos=pos)
        return out
    if op == "attend":
        out = torch.empty_like(st["q"], dtype=torch.float64)
        weight = st["weight"].double() if "weight" in st else None
        for b, n in enumerate(st["lens"]):
            o, s = _exact_attention(st, b, st["q"][b:b + 1], n - 1, n, case["window"], case["sinks"])
            out[b] = o[0]
            if weight is not None:
                weight[b, :, :n] += s
        return out if weight is None else dict(out=out, weight=weight)
    out = torch.empty_like(st["q"], dtype=torch.float64)
    at = 0
    for b, (new, total) in enumerate(zip(st["new"], st["lens"])):
        out[at:at + new] = _exact_attention(st, b, st["q"][at:at + new], total - new, total, case["window"],
                                            case["sinks"])[0]
        at += new
    return out
