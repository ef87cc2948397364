"""Workloads of the multi-request serving operators, with their plain forms.

Three operators that a batch of different requests needs beside the shared
decode step:

* ``shared_prefix_attention``: GQA attention of a batch whose sequences share a
  prefix (a system prompt, a document, a few-shot preamble) held once, followed
  by each sequence's own static cache strip;
* ``lora_delta``: the low-rank adapter of each request beside a projection that
  all of them share;
* ``constrained_argmax``: penalties for repeated tokens, biases and grammar
  masks on the logits, then the greedy pick.

``run`` makes the framework's calls where ``own`` is true and computes the same
from elementary torch operations in 32 bits where it is false.  Sizes are those
of the decode, verify and prompt steps of the stack's geometries (32 or 16
query heads over 8 kv heads of 128 dims, hidden 2560, vocabulary 151936) and
odd ones around them.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
D = 128
WORKSPACE = 48 << 20


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _attention(name, batch, q_len, hq, hkv, prefix, past_lo, past_hi, slots):
    return {"name": name, "op": "attention", "batch": batch, "q_len": q_len, "hq": hq, "hkv": hkv, "prefix": prefix,
            "past_lo": past_lo, "past_hi": past_hi, "slots": slots}


def _lora(name, batch, q_len, k, n, rank, adapters, active, bare):
    return {"name": name, "op": "lora", "batch": batch, "q_len": q_len, "k": k, "n": n, "rank": rank,
            "adapters": adapters, "active": active, "bare": bare}


def _logits(name, batch, vocab, allowed, history, biases, dtype, write):
    return {"name": name, "op": "logits", "batch": batch, "vocab": vocab, "allowed": allowed, "history": history,
            "biases": biases, "dtype": dtype, "write": write}


def listed():
    return [
        # two chats over a short system prompt: latency
        _attention("prefix_b2_p300", 2, 1, 32, 8, 300, 5, 40, 64),
        # the batched decode step: 32 requests over one long system prompt, answers under way
        _attention("prefix_b32_p8192", 32, 1, 32, 8, 8192, 40, 700, 1024),
        # speculative verify of five tokens per request, ragged, an odd prefix, the small model's heads
        _attention("prefix_b13_q5_p5003", 13, 5, 16, 8, 5003, 3, 900, 1027),
        # the requests' own prompts going in behind a shared document
        _attention("prefix_b6_q384_p8192", 6, 384, 32, 8, 8192, 0, 130, 768),
        # one request with an adapter: the QKV projection of one token
        _lora("lora_b1_qkv_r16", 1, 1, 2560, 6144, 16, 4, 1, 0),
        # 32 requests, 20 adapters in use, some requests without one: the gate / up projection
        _lora("lora_b32_gate_up_r16", 32, 1, 2560, 19456, 16, 32, 20, 5),
        # verify of 16 requests x 5 tokens, high rank, the down projection
        _lora("lora_b16_q5_down_r64", 16, 5, 9728, 2560, 64, 12, 9, 1),
        # prompts of 7 requests going in together, odd length
        _lora("lora_b7_q701_qkv_r32", 7, 701, 2560, 6144, 32, 8, 5, 1),
        # one request, free text: penalties and a few biases
        _logits("logits_b1", 1, 151936, 151936, 700, 4, "bfloat16", False),
        # 32 requests in structured output: the grammar leaves a few hundred tokens
        _logits("logits_b32_grammar", 32, 151936, 300, 1500, 0, "bfloat16", False),
        # the largest batch, a mask that bans some tokens, biases, processed logits for a sampler
        _logits("logits_b128_write", 128, 151936, 140000, 2000, 60, "bfloat16", True),
        # an odd vocabulary in fp32 logits
        _logits("logits_b19_odd_f32", 19, 50263, 30011, 311, 9, "float32", True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(("attention", "lora", "logits"))
    if op == "attention":
        hq, hkv = rng.choice(((32, 8), (16, 8), (8, 2), (5, 5)))
        kind = rng.choice(("decode", "decode", "verify", "prompt"))
        if kind == "decode":
            batch, q_len, prefix = _log_int(rng, 1, 96), 1, _log_int(rng, 16, 24000)
        elif kind == "verify":
            batch, q_len, prefix = _log_int(rng, 1, 24), rng.randint(2, 8), _log_int(rng, 16, 12000)
        else:
            batch, q_len, prefix = rng.randint(1, 4), _log_int(rng, 17, 384), _log_int(rng, 16, 8192)
        past_hi = _log_int(rng, 1, 700)
        c = _attention("", batch, q_len, hq, hkv, prefix, rng.randint(0, past_hi), past_hi,
                       past_hi + q_len + rng.randint(0, 60))
    elif op == "lora":
        kind = rng.choice(("decode", "decode", "prompt"))
        if kind == "decode":
            batch = _log_int(rng, 1, 100)
            q_len = 1 if rng.random() < 0.6 else rng.randint(1, max(1, min(6, 128 // batch)))
        else:
            batch, q_len = rng.randint(1, 6), _log_int(rng, 30, 700)
        active = rng.randint(1, 24)
        c = _lora("", batch, q_len, 8 * _log_int(rng, 32, 1216), 8 * _log_int(rng, 16, 768 if kind == "prompt" else 2432),
                  8 * rng.randint(1, 8), active + rng.randint(0, 5), active, rng.randint(0, batch // 4))
    else:
        vocab = _log_int(rng, 1000, 160000)
        batch = _log_int(rng, 1, 100)
        c = _logits("", batch, vocab, rng.choice((vocab, _log_int(rng, 1, vocab), min(vocab, _log_int(rng, 1, 500)))),
                    _log_int(rng, 1, 3000), rng.choice((0, rng.randint(1, 80))), rng.choice(("bfloat16", "float32")),
                    rng.random() < 0.5)
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _pasts(case):
    """Cached positions of the sequences: evenly spread over the case's range."""
    n, lo, hi = case["batch"], case["past_lo"], case["past_hi"]
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _ids(case):
    """Adapter of each sequence: the active ones in turn, the last `bare` sequences without one (-1)."""
    n = case["batch"] - case["bare"]
    return [i % case["active"] for i in range(n)] + [-1] * case["bare"]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    pick = random.Random(seed)

    def normal(shape, std=1.0, dtype=torch.bfloat16):
        return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).mul_(std).to(dtype)

    if case["op"] == "attention":
        b, q, hq, hkv, p, s = (case[k] for k in ("batch", "q_len", "hq", "hkv", "prefix", "slots"))
        past = _pasts(case)
        pick.shuffle(past)
        st = {"q": normal((b * q, hq, D)), "k_prefix": normal((hkv, p, D)), "v_prefix": normal((hkv, p, D)),
              "k_cache": normal((b, hkv, s, D)), "v_cache": normal((b, hkv, s, D)),
              "cache_pos": torch.tensor(past, device=DEV, dtype=torch.int32), "scale": D ** -0.5,
              "out": torch.empty((b * q, hq * D), device=DEV, dtype=torch.bfloat16)}
    elif case["op"] == "lora":
        b, q, k, n, r, a = (case[x] for x in ("batch", "q_len", "k", "n", "rank", "adapters"))
        names = list(range(a))
        pick.shuffle(names)
        ids = [names[i] if i >= 0 else -1 for i in _ids(case)]
        pick.shuffle(ids)
        st = {"x": normal((b * q, k)), "a": normal((a, r, k), k ** -0.5), "b": normal((a, n, r), r ** -0.5),
              "scaling": torch.tensor([pick.choice((0.5, 1.0, 2.0)) for _ in range(a)], device=DEV),
              "adapter_ids": torch.tensor(ids, device=DEV, dtype=torch.int32),
              "out": torch.empty((b * q, n), device=DEV, dtype=torch.float32)}
    else:
        b, v = case["batch"], case["vocab"]
        words = (v + 31) // 32
        tokens = torch.rand((b, case["history"]), generator=g, device=DEV).square_().mul_(v).long()  # frequent ones repeat
        counts = torch.zeros((b, v), device=DEV, dtype=torch.int32)
        half = case["history"] // 2  # the prompt's half counts as seen, the answer's half is counted too
        counts.scatter_add_(1, tokens[:, half:], torch.ones_like(tokens[:, half:], dtype=torch.int32))
        seen = torch.zeros((b, v), device=DEV, dtype=torch.bool).scatter_(1, tokens, True)
        allowed = None
        if case["allowed"] < v:
            keep = torch.rand((b, v), generator=g, device=DEV).topk(case["allowed"], dim=1).indices
            allowed = _pack(torch.zeros((b, v), device=DEV, dtype=torch.bool).scatter_(1, keep, True), words)
        nb = case["biases"]
        st = {"logits": normal((b, v), 3.0, getattr(torch, case["dtype"])), "counts": counts,
              "seen": _pack(seen, words), "allowed": allowed,
              "repetition": torch.empty(b, device=DEV).uniform_(1.0, 1.5, generator=g),
              "frequency": torch.empty(b, device=DEV).uniform_(0.0, 0.5, generator=g),
              "presence": torch.empty(b, device=DEV).uniform_(0.0, 1.0, generator=g),
              "bias_ids": (torch.rand((b, nb), generator=g, device=DEV) * v).int() if nb else None,
              "bias_values": normal((b, nb), 5.0, torch.float32) if nb else None,
              "out_ids": torch.empty(b, device=DEV, dtype=torch.int64),
              "out_logits": torch.empty((b, v), device=DEV) if case["write"] else None}
    st["case"] = dict(case)
    # what a serving program sets aside once: zero-filled scratch that calls share, as the framework's other kernels take it
    st["workspace"] = torch.zeros(WORKSPACE, device=DEV, dtype=torch.uint8)
    return st


def _pack(bits, words):
    """Truth values [b, v] as int32 words [b, words], bit j of word w for index 32 w + j."""
    b, v = bits.shape
    full = torch.zeros((b, words * 32), device=bits.device, dtype=torch.int64)
    full[:, :v] = bits
    w = (full.view(b, words, 32) << torch.arange(32, device=bits.device)).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if case["op"] == "attention":
        return _own_attention(state, case) if own else _plain_attention(state, case)
    if case["op"] == "lora":
        return _own_lora(state, case) if own else _plain_lora(state, case)
    return _own_logits(state) if own else _plain_logits(state)


def _own_attention(st, c):
    from leanstack_b200 import kernels as K

    return K.shared_prefix_attention(st["q"], st["k_prefix"], st["v_prefix"], st["k_cache"], st["v_cache"], c["batch"],
                                     c["q_len"], c["hq"], c["hkv"], D, c["prefix"], c["slots"], st["scale"],
                                     cache_pos=st["cache_pos"], out=st["out"], workspace=st["workspace"])


def _own_lora(st, c):
    from leanstack_b200 import kernels as K

    return K.lora_delta(st["x"], st["a"], st["b"], st["scaling"], st["adapter_ids"], c["q_len"], out=st["out"],
                        workspace=st["workspace"])


def _own_logits(st):
    from leanstack_b200 import kernels as K

    ids = K.constrained_argmax(st["logits"], counts=st["counts"], seen=st["seen"], repetition=st["repetition"],
                               frequency=st["frequency"], presence=st["presence"], bias_ids=st["bias_ids"],
                               bias_values=st["bias_values"], allowed=st["allowed"], record=True,
                               out_ids=st["out_ids"], out_logits=st["out_logits"])
    return {"ids": ids, "logits": st["out_logits"], "counts": st["counts"], "seen": st["seen"]}


def _plain_attention(st, c):
    b, q, hq, hkv, s = c["batch"], c["q_len"], c["hq"], c["hkv"], c["slots"]
    g = hq // hkv
    rows = st["q"].float().view(b, q, hkv, g, D).permute(2, 0, 1, 3, 4) * st["scale"]  # [hkv, b, q, g, D]
    sp = rows.reshape(hkv, b * q * g, D) @ st["k_prefix"].float().transpose(1, 2)
    own_rows = rows.permute(1, 0, 2, 3, 4).reshape(b, hkv, q * g, D)
    sc = (own_rows @ st["k_cache"].float().transpose(2, 3)).view(b, hkv, q, g, s)
    last = st["cache_pos"].long()[:, None] + torch.arange(q, device=DEV)
    hidden = torch.arange(s, device=DEV) > last[..., None]  # [b, q, s]
    sc = sc.masked_fill(hidden[:, None, :, None], float("-inf")).view(b, hkv, q * g, s)
    sp = sp.view(hkv, b, q * g, c["prefix"]).transpose(0, 1)
    m = torch.maximum(sp.amax(-1, keepdim=True), sc.amax(-1, keepdim=True))
    pp, pc = (sp - m).exp(), (sc - m).exp()
    total = pp.sum(-1, keepdim=True) + pc.sum(-1, keepdim=True)
    op = pp.transpose(0, 1).reshape(hkv, b * q * g, c["prefix"]) @ st["v_prefix"].float()
    o = op.view(hkv, b, q * g, D).transpose(0, 1) + pc @ st["v_cache"].float()
    o = (o / total).view(b, hkv, q, g, D).permute(0, 2, 1, 3, 4)
    return o.reshape(b * q, hq * D).to(torch.bfloat16)


def _plain_lora(st, c):
    b, q = c["batch"], c["q_len"]
    ids = st["adapter_ids"].long()
    at = ids.clamp(min=0)
    u = st["x"].float().view(b, q, -1) @ st["a"][at].float().transpose(1, 2)
    y = (u @ st["b"][at].float().transpose(1, 2)) * st["scaling"][at][:, None, None]
    return torch.where((ids >= 0)[:, None, None], y, 0.0).view(b * q, -1)


def _unpack(words, v):
    return ((words[:, :, None] >> torch.arange(32, device=words.device, dtype=torch.int32)) & 1).flatten(1)[:, :v] != 0


def _plain_logits(st):
    x = st["logits"].float()
    v = x.shape[1]
    rep, freq, pres = (st[k][:, None] for k in ("repetition", "frequency", "presence"))
    x = torch.where(_unpack(st["seen"], v), torch.where(x > 0, x / rep, x * rep), x)
    count = st["counts"].float()
    x = torch.where(st["counts"] > 0, (x - freq * count) - pres, x)
    if st["bias_ids"] is not None:
        x = x + torch.zeros_like(x).scatter_add_(1, st["bias_ids"].long(), st["bias_values"])
    ids = torch.arange(v, device=x.device).expand_as(x)
    if st["allowed"] is not None:
        x = torch.where(_unpack(st["allowed"], v), x, float("-inf"))
    best = torch.where(x == x.amax(1, keepdim=True), ids, v).amin(1)
    st["counts"].scatter_add_(1, best[:, None], torch.ones_like(best[:, None], dtype=torch.int32))
    word, bit = best // 32, (best % 32).int()
    old = st["seen"].gather(1, word[:, None])
    st["seen"].scatter_(1, word[:, None], old | (torch.ones_like(bit) << bit)[:, None])
    return {"ids": best, "logits": x if st["out_logits"] is not None else None, "counts": st["counts"],
            "seen": st["seen"]}


# ---------------------------------------------------------------------------
# what one pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] == "attention":
        b, q, hq, hkv, p = (case[k] for k in ("batch", "q_len", "hq", "hkv", "prefix"))
        past = _pasts(case)
        keys = hkv * (p + sum(n + q for n in past))
        pairs = hq * (b * q * p + sum(q * (n + 1) + q * (q - 1) // 2 for n in past))
        return {"bytes": keys * 2 * D * 2 + 2 * b * q * hq * D * 2, "flops": 4 * D * pairs}
    if case["op"] == "lora":
        m, k, n, r = case["batch"] * case["q_len"], case["k"], case["n"], case["rank"]
        ids = [i for i in _ids(case) if i >= 0]
        with_one = len(ids) * case["q_len"]
        return {"bytes": with_one * k * 2 + len(set(ids)) * r * (k + n) * 2 + m * n * 4,
                "flops": 2 * with_one * r * (k + n)}
    b, v = case["batch"], case["vocab"]
    size = 2 if case["dtype"] == "bfloat16" else 4
    masks = v / 8 * (1 if case["allowed"] == v else 2)
    return {"bytes": b * (case["allowed"] * size + masks + (4 * v if case["write"] else 0)), "flops": b * case["allowed"]}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(st, case)
    if case["op"] == "lora":
        x, q = st["x"].double(), case["q_len"]
        out = torch.zeros((x.shape[0], case["n"]), device=DEV, dtype=torch.float64)
        for i, a in enumerate(st["adapter_ids"].tolist()):
            if a >= 0:
                weight = st["b"][a].double() @ st["a"][a].double()
                out[i * q:(i + 1) * q] = st["scaling"][a].double() * torch.nn.functional.linear(x[i * q:(i + 1) * q], weight)
        return out
    if not case["write"]:
        return None  # whole numbers only
    v = case["vocab"]
    out = torch.empty((case["batch"], v), device=DEV, dtype=torch.float64)
    for i in range(case["batch"]):
        row = st["logits"][i].double()
        at = torch.arange(v, device=DEV)

        def bit(words):
            return (words[at // 32].long() >> (at % 32)) % 2 == 1

        known = bit(st["seen"][i])
        theta = st["repetition"][i].double()
        row[known] = torch.where(row[known] < 0, row[known] * theta, row[known] / theta)
        n = st["counts"][i].double()
        row -= n * st["frequency"][i].double() + (n != 0).double() * st["presence"][i].double()
        if st["bias_ids"] is not None:
            row.index_add_(0, st["bias_ids"][i].long(), st["bias_values"][i].double())
        if st["allowed"] is not None:
            row[~bit(st["allowed"][i])] = -math.inf
        out[i] = row
    return {"ids": None, "logits": out, "counts": None, "seen": None}


def _exact_attention(st, c):
    b, q, hq, hkv = c["batch"], c["q_len"], c["hq"], c["hkv"]
    g = hq // hkv
    out = torch.empty((b, q, hq, D), device=DEV, dtype=torch.float64)
    past = st["cache_pos"].tolist()
    qs = st["q"].view(b, q, hq, D)
    for i in range(b):
        n = past[i] + q
        later = torch.ones((q, n), device=DEV, dtype=torch.bool).triu(past[i] + 1)
        later = torch.cat([torch.zeros((q, c["prefix"]), device=DEV, dtype=torch.bool), later], 1)
        for h in range(hkv):
            keys = torch.cat([st["k_prefix"][h], st["k_cache"][i, h, :n]]).double()
            values = torch.cat([st["v_prefix"][h], st["v_cache"][i, h, :n]]).double()
            heads = qs[i, :, h * g:(h + 1) * g].double().transpose(0, 1)  # [g, q, D]
            w = torch.softmax((heads @ keys.T * st["scale"]).masked_fill(later, -math.inf), -1)
            out[i, :, h * g:(h + 1) * g] = (w @ values).transpose(0, 1)
    return out.view(b * q, hq * D)
