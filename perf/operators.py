"""The operators of beam search over the paged cache: what is measured of them, and their plain forms.

Three calls that a decoding step of a beam search makes, in the order it makes them:

  attention   requests of one family (beams of a prompt, requests behind one prefix) read the pages they hold in common once for all
  select      the best continuations over all beams of a request and the whole vocabulary, by the sum of their log probabilities
  copy        rows of the cache move: the page a beam is in the middle of, or the state of a request slot, to the beam that goes on from it

Head counts, layers and the vocabulary are those of the models bench.py runs (SmolLM2-135M / 360M / 1.7B) and of the larger set of layer sizes of the
other designs (16 heads over 2 of 128); pages hold 16 positions unless a case says otherwise.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
# query heads, key-value heads, size of a head
HEADS = {"135M": (9, 3, 64), "360M": (15, 5, 64), "1.7B": (32, 32, 64), "w2048": (16, 2, 128)}
LAYERS = {"135M": 30, "360M": 32, "1.7B": 24}
VOCAB = 49152


def listed():
    return [
        # four beams of a short prompt at the smallest model: launches and latency
        dict(name="attn_135m_4beams", op="attention", model="135M", dtype="bfloat16", page=16, groups=1, members=4, shared=512, own=24, ragged=1),
        # eight beams of the benchmark's prompt at the largest model
        dict(name="attn_1p7b_8beams", op="attention", model="1.7B", dtype="bfloat16", page=16, groups=1, members=8, shared=2048, own=128, ragged=2),
        # six requests with up to five beams each, prompts of different lengths
        dict(name="attn_360m_6x5beams", op="attention", model="360M", dtype="bfloat16", page=16, groups=6, members=5, shared=2048, own=64, ragged=3),
        # a full batch of requests behind one long prefix, answers of different lengths: the largest
        dict(name="attn_1p7b_64_prefix", op="attention", model="1.7B", dtype="bfloat16", page=16, groups=1, members=64, shared=6000, own=700, ragged=4),
        # sixteen requests behind a very long document, wide heads, eight of them to a key-value head
        dict(name="attn_w2048_16_long", op="attention", model="w2048", dtype="bfloat16", page=16, groups=1, members=16, shared=32000, own=300, ragged=5),
        # beams in float32
        dict(name="attn_135m_6beams_f32", op="attention", model="135M", dtype="float32", page=16, groups=1, members=6, shared=1000, own=40, ragged=6),
        # one request, four beams: the smallest selection
        dict(name="select_4", op="select", requests=1, beams=4, vocab=VOCAB, keep=8),
        # three requests of five beams, an odd vocabulary
        dict(name="select_3x5_odd", op="select", requests=3, beams=5, vocab=50257, keep=10),
        # eight requests of eight beams: every slot of a full batch
        dict(name="select_8x8", op="select", requests=8, beams=8, vocab=VOCAB, keep=16),
        # two wide searches over a large vocabulary
        dict(name="select_2x32_wide", op="select", requests=2, beams=32, vocab=131072, keep=64),
        # three of eight beams take over another's unfinished page, in every layer of the smallest model
        dict(name="copy_pages_135m", op="copy", layers=30, rows=512, numbers=2 * 3 * 16 * 64, dtype="bfloat16", moves=3),
        # seven of sixteen slots take over another's matrix states (16 heads of 128 x 128 and a few numbers beside them), in twelve layers
        dict(name="copy_states_w2048", op="copy", layers=12, rows=16, numbers=16 * 128 * 128 + 64, dtype="float32", moves=7),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "select", "select", "copy"])
    if op == "attention":
        model = rng.choice(sorted(HEADS))
        groups = rng.choice([1, 1, rng.randint(2, 8)])
        return dict(op="attention", model=model, dtype=rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"]), page=rng.choice([16, 16, 16, 8, 12, 32, 64]),
                    groups=groups, members=_log(rng, 1, 64 // groups), shared=_log(rng, 16, 32000 if model == "w2048" else 6000), own=_log(rng, 1, 700),
                    ragged=rng.randint(7, 10**6))
    if op == "select":
        beams = _log(rng, 1, 32)
        return dict(op="select", requests=_log(rng, 1, 64 // beams), beams=beams, vocab=rng.choice([VOCAB, _log(rng, 500, 131072)]), keep=rng.choice([2 * beams, rng.randint(1, 64)]))
    if rng.random() < 0.5:
        model = rng.choice(sorted(LAYERS))
        return dict(op="copy", layers=LAYERS[model], rows=64, numbers=2 * HEADS[model][1] * rng.choice([8, 16, 16, 12]) * HEADS[model][2], dtype=rng.choice(["bfloat16", "float32"]),
                    moves=_log(rng, 1, 32))
    return dict(op="copy", layers=rng.randint(1, 12), rows=16, numbers=_log(rng, 1000, 270000), dtype="float32", moves=rng.randint(1, 8))


def _lengths(case):
    """For each family: how many positions its members share (whole pages), and how many each member has of its own (the token it is at counts)."""
    rng, out = random.Random(case["ragged"]), []
    for g in range(case["groups"]):
        members = case["members"] if g == 0 else rng.randint(1, case["members"])
        shared = case["shared"] if g == 0 else rng.randint(case["shared"] // 2, case["shared"])
        out.append((shared // case["page"] * case["page"], [rng.randint(1, case["own"]) for _ in range(members)]))
    return out


def work(case):
    if case["op"] == "attention":
        nh, nkv, hd = HEADS[case["model"]]
        size = 2 if case["dtype"] == "bfloat16" else 4
        lens = _lengths(case)
        tokens = sum(len(own_) for _, own_ in lens)
        cached = sum(shared + sum(own_) for shared, own_ in lens)
        pairs = sum(shared * len(own_) + sum(own_) for shared, own_ in lens)
        return {"bytes": (cached * 2 * nkv + tokens * 2 * nh) * hd * size, "flops": pairs * nh * hd * 4}
    if case["op"] == "select":
        rows = case["requests"] * case["beams"]
        return {"bytes": rows * case["vocab"] * 4 + rows * 4 + case["requests"] * case["keep"] * 12, "flops": rows * case["vocab"] * 3}
    return {"bytes": 2 * case["moves"] * case["layers"] * case["numbers"] * (2 if case["dtype"] == "bfloat16" else 4), "flops": 0}


# -- inputs -------------------------------------------------------------------------------------------------------------------------


class _State:
    pass


def _attention_inputs(case, g):
    """A layer's pages in a random order, every request's block table, the batch's tokens in a random order, and its families."""
    nh, nkv, hd = HEADS[case["model"]]
    page, dtype = case["page"], DTYPES[case["dtype"]]
    lens = _lengths(case)
    need = sum(shared // page + sum(-(-n // page) for n in own_) for shared, own_ in lens)
    s = _State()
    s.op, s.nh, s.nkv, s.hd, s.page, s.scale = "attention", nh, nkv, hd, page, hd ** -0.5
    s.pages = torch.randn((need + 3, 2, nkv, page, hd), generator=g, device="cuda").to(dtype)
    free = torch.randperm(need + 3, generator=g, device="cuda").tolist()
    tokens = sum(len(own_) for _, own_ in lens)
    place = torch.randperm(tokens, generator=g, device="cuda").tolist()       # where in the batch a family's next member stands
    tables, positions, members, starts, shared_lens = [None] * tokens, [0] * tokens, [], [0], []
    for shared, own_ in lens:
        first = [free.pop() for _ in range(shared // page)]
        for n in own_:
            t = place[len(members)]
            members.append(t)
            tables[t] = first + [free.pop() for _ in range(-(-n // page))]
            positions[t] = shared + n - 1
        starts.append(len(members))
        shared_lens.append(shared)
    wide = max(len(t) for t in tables) + 1
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")      # noqa: E731
    s.tables = ints([t + [0] * (wide - len(t)) for t in tables])
    s.positions, s.seg = ints(positions), ints(list(range(tokens)))
    s.members, s.starts, s.shared = ints(members), ints(starts), ints(shared_lens)
    s.q = (torch.randn((tokens, nh * hd), generator=g, device="cuda") * 1.5).to(dtype)
    s.out, s.scratch = torch.empty_like(s.q), None
    return s


def _select_inputs(case, g):
    rows = case["requests"] * case["beams"]
    s = _State()
    s.op, s.beams, s.keep = "select", case["beams"], min(case["keep"], case["beams"] * case["vocab"])
    # most of the vocabulary far below a few hundred likely tokens
    s.logits = torch.randn((rows, case["vocab"]), generator=g, device="cuda") * 2.0
    likely = torch.randint(0, case["vocab"], (rows, min(200, case["vocab"])), generator=g, device="cuda")
    s.logits.scatter_add_(1, likely, torch.rand(likely.shape, generator=g, device="cuda") * 9.0)
    s.scores = -20.0 - 4.0 * torch.rand((rows,), generator=g, device="cuda")
    s.out = tuple(torch.empty((case["requests"], s.keep), dtype=d, device="cuda") for d in (torch.float32, torch.int32, torch.int32))
    s.scratch = None
    return s


def _copy_inputs(case, g):
    s = _State()
    s.op = "copy"
    s.arena = torch.randn((case["layers"], case["rows"], case["numbers"]), generator=g, device="cuda").to(DTYPES[case["dtype"]])
    order = torch.randperm(case["rows"], generator=g, device="cuda").tolist()
    s.dst = order[:case["moves"]]
    s.src = [order[case["moves"] + i // 2] for i in range(case["moves"])]           # two beams go on from one
    s.src_dev, s.dst_dev = (torch.tensor(v, device="cuda") for v in (s.src, s.dst))
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) & 0x7FFFFFFFFFFFFFFF)
    return {"attention": _attention_inputs, "select": _select_inputs, "copy": _copy_inputs}[case["op"]](case, g)


# -- one pass -----------------------------------------------------------------------------------------------------------------------


def _plain_attention(s):
    tokens, blocks = s.q.shape[0], s.tables.shape[1]
    tables = s.tables.long()[s.seg.long()]
    k = s.pages[:, 0][tables].transpose(1, 2).reshape(tokens, s.nkv, blocks * s.page, s.hd).float()
    v = s.pages[:, 1][tables].transpose(1, 2).reshape(tokens, s.nkv, blocks * s.page, s.hd).float()
    q = s.q.view(tokens, s.nkv, s.nh // s.nkv, s.hd).float()
    z = (q @ k.transpose(2, 3)) * s.scale
    hidden = torch.arange(blocks * s.page, device="cuda") > s.positions[:, None]
    z = z.masked_fill(hidden[:, None, None], -math.inf)
    p = torch.exp(z - z.amax(-1, keepdim=True))
    return ((p @ v) / p.sum(-1, keepdim=True)).reshape(tokens, s.nh * s.hd).to(s.q.dtype)


def _plain_select(s):
    x = s.logits.double()
    top = x.amax(1, keepdim=True)
    total = s.scores.double()[:, None] + (x - top - torch.log(torch.exp(x - top).sum(1, keepdim=True)))
    total = total.view(-1, s.beams * x.shape[1])
    best, at = torch.sort(total, dim=1, descending=True, stable=True)
    best, at = best[:, :s.keep], at[:, :s.keep]
    return best.float(), (at // x.shape[1]).int(), (at % x.shape[1]).int()


def _plain_copy(s):
    s.arena[:, s.dst_dev] = s.arena[:, s.src_dev]
    return s.arena


def run(state):
    s = state
    if not own:
        return {"attention": _plain_attention, "select": _plain_select, "copy": _plain_copy}[s.op](s)
    from vitna_anchor_b200 import ops
    if s.op == "attention":
        if s.scratch is None:               # made once, zero at first use, and kept by the program
            s.scratch = torch.zeros(ops.attention_shared_scratch_bytes(s.q.shape[0], s.nh, s.nkv, s.hd), dtype=torch.uint8, device="cuda")
        return ops.attention_shared(s.q, s.pages, s.tables, s.seg, s.positions, s.members, s.starts, s.shared, s.out, s.scratch, s.nh, s.nkv, s.hd, s.scale)
    if s.op == "select":
        if s.scratch is None:
            s.scratch = torch.zeros(ops.beam_select_scratch_bytes(s.logits.shape[0], s.logits.shape[1], s.keep), dtype=torch.uint8, device="cuda")
        return ops.beam_select(s.logits, s.scores, s.beams, s.keep, s.out, s.scratch)
    return ops.copy_rows(s.arena, s.src, s.dst)


# -- the definition, in 64 bits ---------------------------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if s.op == "attention":
        out, reps = [], s.nh // s.nkv
        for t in range(s.q.shape[0]):
            at = torch.arange(int(s.positions[t]) + 1, device="cuda")
            page = s.tables[t].long()[at // s.page]
            kv = s.pages[page, :, :, at % s.page].double()                  # [positions, 2, kv heads, dim]
            k, v = (kv[:, i].repeat_interleave(reps, dim=1) for i in (0, 1))
            z = torch.einsum("phd,hd->hp", k, s.q[t].double().view(s.nh, s.hd)) / math.sqrt(s.hd)
            out.append(torch.einsum("hp,phd->hd", torch.softmax(z, dim=1), v).reshape(-1))
        return torch.stack(out)
    if s.op == "select":
        x, scores = s.logits.cpu().numpy().astype(np.float64), s.scores.cpu().numpy().astype(np.float64)
        logp = x - np.logaddexp.reduce(x, axis=1, keepdims=True)
        best, parent, token = [], [], []
        for r in range(case["requests"]):
            mine = slice(r * s.beams, (r + 1) * s.beams)
            flat = (scores[mine, None] + logp[mine]).reshape(-1)
            order = np.argsort(-flat, kind="stable")[:s.keep]
            best.append(flat[order]), parent.append(order // case["vocab"]), token.append(order % case["vocab"])
        return np.stack(best), np.stack(parent), np.stack(token)
    return None
