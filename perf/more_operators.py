"""Operators of a beam search's step and of the words' rows it goes on with, as cases that can be timed
and compared: the best extensions of an utterance's hypotheses (`extend_beams`), the states that
follow them (`reorder_states`), and the rows of a table of word embeddings, scaled and with dropout,
for single words and in training with the table's gradient (`embed_words`).

A case is a dict; which of the keys it has depends on its task:

    task      "extend", "reorder", "embed" (forward and gradient) or "lookup" (forward alone)
    dtype     "f32" or "bf16": emissions and predictions, states, table
    checked   indices validated by the call (it synchronises) or not (it only enqueues work)
  extend
    B N W V   utterances, hypotheses of each, extensions kept of each, vocabulary
    spread    the hypotheses of an utterance are at so many different frames
    done gone shares of the hypotheses that are finished (no node, but a score) and that are not there
    std       scores are N(0, std); on most frames one word, often the blank, is raised by 4 to 12
  reorder
    B N W     utterances, hypotheses of each before and after
    layers    predictor layers, each with two states of the shape `state` per hypothesis
    state     dimensions of a state, as text: "640" or "100x512"
    history   int32 words remembered per hypothesis (0: none)
  embed, lookup
    B U       words are int32 [B, U]; those beyond an utterance's length (uniform in [u_min, U]) are -1
    R H       rows of the table, numbers in a row
    scale dropout
"""
import math

import torch

own = False


def _extend(B, N, W, V, spread=1, done=0.1, gone=0.05, std=1.5, dtype="f32", checked=False):
    return {"task": "extend", "B": B, "N": N, "W": W, "V": V, "spread": spread, "done": done,
            "gone": gone, "std": std, "dtype": dtype, "checked": checked}


def _reorder(B, N, W, layers, state, history=0, dtype="f32", checked=False):
    return {"task": "reorder", "B": B, "N": N, "W": W, "layers": layers, "state": state,
            "history": history, "dtype": dtype, "checked": checked}


def _embed(task, B, U, R, H, u_min=None, scale=1.0, dropout=0.0, dtype="f32", checked=False):
    return {"task": task, "B": B, "U": U, "R": R, "H": H, "u_min": U if u_min is None else u_min,
            "scale": scale, "dropout": dropout, "dtype": dtype, "checked": checked}


def listed():
    return [dict(case, name=name) for name, case in [
        # a step of a beam search: 8 hypotheses of each of 4 utterances, 1024 word pieces and a blank
        ("extend_step_v1025", _extend(4, 8, 8, 1025, spread=3)),
        # one utterance while a user waits, large vocabulary
        ("extend_one_v32000", _extend(1, 8, 8, 32000, done=0.0, gone=0.0)),
        # a batch of utterances on a server, mixed-precision model, all hypotheses at one frame
        ("extend_step_v4096_bf16", _extend(64, 16, 16, 4096, dtype="bf16", checked=True)),
        # the widest search over the largest batch and vocabulary
        ("extend_wide_v32000", _extend(64, 32, 32, 32000, spread=4)),
        # two LSTM layers and the words so far of 4 x 8 hypotheses
        ("reorder_lstm_small", _reorder(4, 8, 8, 2, "640", history=100)),
        # a batch whose beams grow from 16 to 24, rows of an odd length
        ("reorder_batch_odd_bf16", _reorder(64, 16, 24, 2, "641", history=77, dtype="bf16",
                                            checked=True)),
        # keys and values of a predictor with attention: 100 labels of 512 numbers in two layers
        ("reorder_cache_bf16", _reorder(32, 16, 16, 2, "100x512", dtype="bf16")),
        # the smallest training step: two transcripts over a character set
        ("embed_tiny_r30", _embed("embed", 2, 11, 30, 128, u_min=2, dropout=0.1, checked=True)),
        # a predictor's inputs for a batch of 32 transcripts of 100 labels
        ("embed_r10000_h640", _embed("embed", 32, 101, 10000, 640, u_min=61, scale=math.sqrt(640),
                                     dropout=0.1)),
        # the predictions themselves, from the word before: a table of 1025 rows of 1025 scores
        ("embed_bigram_v1025", _embed("embed", 16, 81, 1025, 1025, u_min=21)),
        # the largest batch and table, mixed precision
        ("embed_r32000_h1024_bf16", _embed("embed", 256, 201, 32000, 1024, u_min=121,
                                           dropout=0.2, dtype="bf16")),
        # the words that a step of 64 x 16 hypotheses has chosen
        ("lookup_step_bf16", _embed("lookup", 64, 16, 32000, 640, scale=math.sqrt(640),
                                    dtype="bf16")),
    ]]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another case of the same ranges: 1-64 utterances of 1-64 hypotheses, 28-32000 words (half of
    the vocabularies a multiple of 8); 1-4 layers of 16-2048 numbers, or of 1-200 labels of them; up to
    256 transcripts of 1-201 labels, tables of 28-32000 rows of 16-2048 numbers."""
    while True:
        task = rng.choice(["extend", "extend", "reorder", "reorder", "embed", "embed", "embed", "lookup"])
        dtype = rng.choice(["f32", "bf16"])
        checked = rng.random() < 0.3
        if task == "extend":
            V = _log(rng, 28, 32000)
            if rng.random() < 0.5:
                V = (V + 7) // 8 * 8
            B, N, W = _log(rng, 1, 64), _log(rng, 1, 64), _log(rng, 1, 64)
            if B * N * V > 6.5e7:
                continue
            return _extend(B, N, W, V, spread=rng.choice([1, 1, 3, 6]),
                           done=rng.choice([0.0, 0.1, 0.3]), gone=rng.choice([0.0, 0.05]),
                           std=rng.choice([1.0, 1.5, 2.0]), dtype=dtype, checked=checked)
        if task == "reorder":
            B, N, layers = _log(rng, 1, 64), _log(rng, 1, 32), rng.randint(1, 4)
            W = N if rng.random() < 0.5 else _log(rng, 1, 32)
            H, L = _log(rng, 16, 2048), rng.choice([0, 0, 1]) * _log(rng, 1, 200)
            if rng.random() < 0.6:
                H = (H + 7) // 8 * 8
            if B * max(N, W) * layers * 2 * H * max(L, 1) * (2 if dtype == "bf16" else 4) > 2.0e8:
                continue
            return _reorder(B, N, W, layers, "%dx%d" % (L, H) if L else "%d" % H,
                            history=rng.choice([0, 1]) * _log(rng, 1, 200), dtype=dtype,
                            checked=checked)
        if task == "lookup":
            B, U = _log(rng, 1, 64), _log(rng, 1, 32)
        else:
            B, U = _log(rng, 1, 256), _log(rng, 1, 201)
        R, H = _log(rng, 28, 32000), _log(rng, 16, 2048)
        if rng.random() < 0.6:
            H = (H + 7) // 8 * 8
        if (2 * B * U + 2 * R) * H * (2 if dtype == "bf16" else 4) > 3.4e8:
            continue
        return _embed(task, B, U, R, H, u_min=max(1, int(U * rng.uniform(0.3, 1.0))),
                      scale=rng.choice([1.0, math.sqrt(H)]),
                      dropout=rng.choice([0.0, 0.1, 0.3]) if task == "embed" else 0.0, dtype=dtype,
                      checked=checked)


def _type(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    state = {"case": case}
    {"extend": _prepare_extend, "reorder": _prepare_reorder, "embed": _prepare_embed,
     "lookup": _prepare_embed}[case["task"]](case, g, state)
    return state


def _prepare_extend(case, g, state):
    dev, B, N, V, T = "cuda", case["B"], case["N"], case["V"], case["spread"] + 3
    E = torch.empty((B, T, V), device=dev).normal_(0.0, case["std"], generator=g)
    word = torch.randint(0, V, (B, T, 1), generator=g, device=dev)
    word[torch.rand((B, T, 1), generator=g, device=dev) < 0.5] = 0
    by = 4 + 8 * torch.rand((B, T, 1), generator=g, device=dev)
    by[torch.rand((B, T, 1), generator=g, device=dev) < 0.2] = 0
    E.scatter_add_(2, word, by)
    P = torch.empty((B, N, V), device=dev).normal_(0.0, case["std"] / 2, generator=g)
    first = torch.randint(0, 4, (B, 1), generator=g, device=dev)
    frames = first + torch.randint(0, case["spread"], (B, N), generator=g, device=dev)
    positions = torch.arange(N, device=dev).expand(B, N)
    kind = torch.rand((B, N), generator=g, device=dev)
    scores = -40.0 + 4.0 * torch.randn((B, N), generator=g, device=dev)
    scores = torch.where(kind < case["gone"], -math.inf, scores)
    none = (kind >= case["gone"]) & (kind < case["gone"] + case["done"])
    frames, positions = torch.where(none, -1, frames), torch.where(none, -1, positions)
    state.update(E=E.to(_type(case)), P=P.to(_type(case)), frames=frames.int().contiguous(),
                 positions=positions.int().contiguous(), scores=scores)


def _prepare_reorder(case, g, state):
    dev, B, N = "cuda", case["B"], case["N"]
    shape = [B, N] + [int(n) for n in case["state"].split("x")]
    states = [torch.empty(shape, device=dev).normal_(generator=g).to(_type(case))
              for _ in range(2 * case["layers"])]
    if case["history"]:
        states.append(torch.randint(0, 32000, (B, N, case["history"]), generator=g, device=dev).int())
    # the best hypotheses have several successors, many of the others none
    parents = (torch.rand((B, case["W"]), generator=g, device=dev) ** 1.5 * N).int().clamp(max=N - 1)
    state.update(states=states, parents=parents)


def _prepare_embed(case, g, state):
    dev, B, U, R, H = "cuda", case["B"], case["U"], case["R"], case["H"]
    table = torch.empty((R, H), device=dev).normal_(generator=g).to(_type(case))
    # words as frequent as in running text (the n-th of them 1 / n), the start symbol, padding
    words = (torch.exp(torch.rand((B, U), generator=g, device=dev) * math.log(R)) - 1.0).long()
    words = words.clamp(max=R - 1)
    if case["task"] == "embed":
        words[:, 0] = 0
        lengths = torch.randint(case["u_min"], U + 1, (B, 1), generator=g, device=dev)
        lengths[0] = U
        words = torch.where(torch.arange(U, device=dev) < lengths, words, -1)
        table.requires_grad_(True)
        state["deltas"] = torch.empty((B, U, H), device=dev).normal_(generator=g).to(_type(case))
    state.update(table=table, words=words.int(),
                 seed=torch.randint(0, 2 ** 62, (1,), generator=g, device=dev))


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    with torch.no_grad():
        if case["task"] == "extend":
            return _plain_extend(case, state)
        if case["task"] == "reorder":
            return _plain_reorder(state)
        return _plain_embed(case, state)


def _run_own(case, state):
    import transducer_b200
    if case["task"] == "extend":
        scores, parents, words = transducer_b200.extend_beams(
            state["E"], state["P"], state["frames"], state["positions"], state["scores"], case["W"],
            validate_nodes=case["checked"])
        return {"scores": scores, "parents": parents, "words": words}
    if case["task"] == "reorder":
        return transducer_b200.reorder_states(state["states"], state["parents"],
                                              validate_parents=case["checked"])
    dropout = {"dropout": case["dropout"], "seed": state["seed"]} if case["dropout"] else {}
    rows = transducer_b200.embed_words(state["table"], state["words"], scale=case["scale"],
                                       validate_words=case["checked"], **dropout)
    if case["task"] == "lookup":
        return rows
    grad, = torch.autograd.grad(rows, state["table"], state["deltas"])
    return {"rows": rows.detach(), "grad": grad}


def _plain_extend(case, state):
    """In 64 bits: which extensions are the best is a comparison of long sums."""
    E, P, W, V = state["E"], state["P"], case["W"], case["V"]
    frames, positions, scores = state["frames"], state["positions"], state["scores"]
    b = torch.arange(E.shape[0], device=E.device)[:, None]
    z = E[b, frames.clamp(min=0).long()].float() + P[b, positions.clamp(min=0).long()].float()
    none = (frames < 0) | (positions < 0)
    z = z.double()
    best = z.amax(-1, keepdim=True)
    lse = best + (z - best).exp().sum(-1, keepdim=True).log()
    z = scores[..., None].double() + (z - lse)
    z = z.masked_fill_(none[..., None], -math.inf)
    stay = scores.double().masked_fill(~none, -math.inf)
    # a hypothesis' own place comes before its extensions
    z = torch.cat((stay[..., None], z), -1).flatten(1)
    if W > z.shape[1]:
        z = torch.nn.functional.pad(z, (0, W - z.shape[1]), value=-math.inf)
    z, at = z.sort(dim=1, descending=True, stable=True)
    z, at = z[:, :W], at[:, :W]
    left = z == -math.inf
    return {"scores": z.float(), "parents": (at // (V + 1)).int().masked_fill(left, -1),
            "words": (at % (V + 1) - 1).int().masked_fill(left, -1)}


def _plain_reorder(state):
    parents = state["parents"].long()
    b = torch.arange(parents.shape[0], device=parents.device)[:, None]
    return [s[b, parents] for s in state["states"]]


def _philox(counter, key):
    """Philox4x32-10 (Salmon, Moraes, Dror and Shaw, 2011): four 32-bit numbers, in int64, of each counter."""
    low = 0xffffffff
    c0, c1, c2, c3 = counter
    k0, k1 = key
    for _ in range(10):
        a, b = c0 * 0xd2511f53, c2 * 0xcd9e8d57   # (64 bits that wrap hold both halves)
        c0, c1, c2, c3 = (b >> 32 & low) ^ c1 ^ k0, b & low, (a >> 32 & low) ^ c3 ^ k1, a & low
        k0, k1 = k0 + 0x9e3779b9 & low, k1 + 0xbb67ae85 & low
    return c0, c1, c2, c3


def _threshold(case):
    return round(case["dropout"] * 65536)


def _kept(case, n, H, seed):
    """Which numbers of the rows `n` stay: 16 bits of the generator are at least 65536 dropout."""
    group = torch.arange((H + 7) // 8, device=n.device)
    counter = torch.broadcast_tensors(n[:, None] & 0xffffffff, n[:, None] >> 32, group, group * 0)
    bits = torch.stack(_philox(counter, (seed & 0xffffffff, seed >> 32 & 0xffffffff)), -1)
    bits = torch.stack((bits & 0xffff, bits >> 16), -1).flatten(1)[:, :H]
    return bits >= _threshold(case)


def _plain_embed(case, state):
    table, words = state["table"], state["words"].flatten().long()
    factor = case["scale"] * 65536 / (65536 - _threshold(case))
    here = (words >= 0)[:, None]
    if case["dropout"]:
        here = here & _kept(case, torch.arange(words.numel(), device=words.device), case["H"],
                            state["seed"])
    at = words.clamp(min=0)
    rows = torch.where(here, table[at].float() * factor, 0.0)
    rows = rows.to(table.dtype).view(case["B"], case["U"], case["H"])
    if case["task"] == "lookup":
        return rows
    grad = torch.zeros(table.shape, device=table.device)
    grad.index_add_(0, at, torch.where(here, state["deltas"].flatten(0, 1).float(), 0.0))
    return {"rows": rows, "grad": (grad * factor).to(table.dtype)}


def work(case):
    """Every row that is needed read once, every output written once (the table's gradient whole).  Per
    word of a hypothesis: the sum of the scores, an exponential and its sum, a comparison; per
    number of an embedding: the factor, and in the gradient a sum."""
    size = 2 if case["dtype"] == "bf16" else 4
    B = case["B"]
    if case["task"] == "extend":
        live = case["N"] * (1.0 - case["done"] - case["gone"])
        frames = case["spread"] * (1.0 - (1.0 - 1.0 / case["spread"]) ** live) if live else 0.0
        return {"bytes": B * (size * case["V"] * (max(frames, 1.0) + live) + 12.0 * (case["N"] + case["W"])),
                "flops": 4.0 * B * live * case["V"]}
    if case["task"] == "reorder":
        row = size * 2 * case["layers"] * math.prod(int(n) for n in case["state"].split("x"))
        row += 4 * case["history"]
        # (parents are N u^1.5: the n-th hypothesis has one of W successors with this probability)
        N, W = case["N"], case["W"]
        share = [((n + 1) / N) ** (2 / 3) - (n / N) ** (2 / 3) for n in range(N)]
        read = sum(1.0 - (1.0 - p) ** W for p in share)
        return {"bytes": B * (row * (read + W) + 4.0 * W), "flops": 0.0}
    R, H, U = case["R"], case["H"], case["U"]
    words = B * U if case["task"] == "lookup" else U + (B - 1) * (case["u_min"] + U) / 2
    share = [math.log((n + 2) / (n + 1)) / math.log(R) for n in range(R - 1)]
    read = sum(1.0 - (1.0 - p) ** words for p in share)
    nbytes = size * H * (read + B * U) + 4.0 * B * U
    if case["task"] == "lookup":
        return {"bytes": nbytes, "flops": float(B * U * H)}
    return {"bytes": nbytes + size * H * (words + R), "flops": 3.0 * B * U * H}


def exact(case, seed):
    """The same from the definitions in 64 bits."""
    state = prepare(case, seed)
    if case["task"] == "extend":
        return {"scores": _exact_extend(case, state), "parents": None, "words": None}
    if case["task"] == "reorder":
        picked = []
        for s in state["states"]:
            one = [s[b].index_select(0, state["parents"][b].long()) for b in range(case["B"])]
            picked.append(torch.stack(one))
        return picked
    return _exact_embed(case, state)


def _exact_extend(case, state):
    out = []
    for b in range(case["B"]):
        candidates = []
        for n in range(case["N"]):
            t, u = state["frames"][b, n].item(), state["positions"][b, n].item()
            score = state["scores"][b, n].double()
            if t < 0 or u < 0:
                candidates.append(score[None])
                continue
            # (the scores of a node are sums in 32 bits by definition)
            z = (state["E"][b, t].float() + state["P"][b, u].float()).double()
            row = torch.log_softmax(z, 0).topk(min(case["W"], case["V"])).values
            candidates.append(score + row)
        best = torch.cat(candidates).sort(descending=True).values[:case["W"]]
        fill = torch.full((case["W"] - best.numel(),), -math.inf, dtype=best.dtype, device=best.device)
        out.append(torch.cat((best, fill)))
    return torch.stack(out)


def _times(a, m):
    """High and low 32 bits of a * m, both below 2^32, from products of halves."""
    a0, a1, m0, m1 = a % 65536, a // 65536, m % 65536, m // 65536
    low = a0 * m0
    mid = a1 * m0 + low // 65536
    mid2 = a0 * m1 + mid % 65536
    return a1 * m1 + mid // 65536 + mid2 // 65536, mid2 % 65536 * 65536 + low % 65536


def _exact_embed(case, state):
    table, H, R = state["table"].detach(), case["H"], case["R"]
    words = state["words"].flatten().long()
    factor = case["scale"] / (1.0 - _threshold(case) / 65536)
    rows, sums = [], torch.zeros((R, H), dtype=torch.float64, device=table.device)
    for first in range(0, words.numel(), 4096):
        n = torch.arange(first, min(first + 4096, words.numel()), device=words.device)
        kept = torch.ones((n.numel(), H), dtype=torch.float64, device=words.device)
        if case["dropout"]:
            h = torch.arange(0, H, 8, device=n.device)
            x = [n[:, None] % 2 ** 32 + 0 * h, n[:, None] // 2 ** 32 + 0 * h, h // 8 + 0 * n[:, None],
                 0 * h + 0 * n[:, None]]
            key = [state["seed"].item() % 2 ** 32, state["seed"].item() // 2 ** 32 % 2 ** 32]
            for turn in range(10):
                k = [(key[0] + turn * 0x9e3779b9) % 2 ** 32, (key[1] + turn * 0xbb67ae85) % 2 ** 32]
                (p, q), (r, s) = _times(x[0], 0xd2511f53), _times(x[2], 0xcd9e8d57)
                x = [r ^ x[1] ^ k[0], s, p ^ x[3] ^ k[1], q]
            for j in range(8):
                number = x[j // 2] // 65536 ** (j % 2) % 65536
                kept[:, j::8] = (number >= _threshold(case)).double()[:, :kept[:, j::8].shape[1]]
        kept[words[n] < 0] = 0.0
        at = words[n].clamp(min=0)
        rows.append(table[at].double() * kept * factor)
        if case["task"] == "embed":
            sums.index_put_((at,), state["deltas"].flatten(0, 1)[n].double() * kept, accumulate=True)
    rows = torch.cat(rows).view(case["B"], case["U"], H)
    return rows if case["task"] == "lookup" else {"rows": rows, "grad": sums * factor}
