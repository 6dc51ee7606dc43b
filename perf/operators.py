"""Operators on single nodes of the transducer's lattice, as cases that can be timed and compared:
the best words of a node with what is left of its distribution (`top_words`), distillation from a
teacher's recorded best words, forward and backward (`NodeDistillationLoss`), and drawing a word
from given random numbers (`sample_words`).

Node n of utterance b is frame frames[b, n] and label position positions[b, n] (both int32
[B, N], -1: no node there); its scores are z[v] = E[b, frame, v] + P[b, position, v], summed in 32
bits.  A case is a dict:

    task      "top", "distill" or "sample"
    B T U V   utterances, frames, longest transcript (predictions have U + 1 rows), vocabulary
    nodes     "path": one way through the lattice of each utterance, a node for each blank and each
              label (N = T + U); "lattice": all T * (U + 1) nodes, frame by frame; "step": `N` nodes
              of one frame per utterance (hypotheses that are extended now), node n at position n
    t_min u_min  lengths of the utterances are uniform in [t_min, T] and [u_min, U]
    K         words listed per node (top, distill)
    rest      distill: whether the teacher's record says how much the words beyond the K best weigh
    temperature  divides the scores
    top_k top_p min_p  sample: 0, 1.0 and 0.0 switch them off
    std       scores are N(0, std); on most frames one word, often the blank, is raised by 4 to 12
    dtype     "f32" or "bf16" storage of emissions, predictions and their gradients
    checked   nodes validated by the call (it synchronises) or not (it only enqueues work)
"""
import math

import torch

own = False


def _case(name, task, B, T, U, V, nodes, t_min=None, u_min=None, N=0, K=0, rest=False,
          temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, std=1.5, dtype="f32", checked=False):
    case = {"task": task, "B": B, "T": T, "U": U, "V": V, "nodes": nodes,
            "t_min": T if t_min is None else t_min, "u_min": U if u_min is None else u_min,
            "N": N, "K": K, "rest": rest, "temperature": temperature, "top_k": top_k,
            "top_p": top_p, "min_p": min_p, "std": std, "dtype": dtype, "checked": checked}
    if name is not None:
        case["name"] = name
    return case


def listed():
    return [
        # a step of a beam search: 8 hypotheses of each of 4 utterances, 1024 word pieces and a blank
        _case("top_beam_v1025", "top", 4, 300, 7, 1025, "step", N=8, K=8),
        # every node of small lattices (a teacher whose record is not bound to one alignment)
        _case("top_lattice_v512", "top", 8, 150, 30, 512, "lattice", t_min=75, u_min=10, K=16,
              checked=True),
        # a teacher's record along the alignments of a batch of long utterances
        _case("top_path_v10000_bf16", "top", 8, 2000, 100, 10000, "path", t_min=1500, u_min=60,
              K=32, temperature=2.0, dtype="bf16"),
        # the smallest training step: two short utterances over a character set
        _case("distill_tiny_v30", "distill", 2, 50, 10, 30, "path", t_min=25, u_min=1, K=4,
              checked=True),
        # a small word-piece vocabulary on long utterances, with the rest's weight recorded
        _case("distill_path_v1000", "distill", 8, 2000, 100, 1000, "path", K=16, rest=True),
        # ragged mid-sized utterances, rows of an odd length, softened distributions
        _case("distill_path_v1025_odd", "distill", 16, 600, 80, 1025, "path", t_min=250, u_min=20,
              K=16, temperature=2.0, checked=True),
        # every node of small lattices
        _case("distill_lattice_v512", "distill", 4, 100, 20, 512, "lattice", t_min=50, u_min=10,
              K=8, rest=True),
        # a large batch over a large vocabulary from a mixed-precision model
        _case("distill_path_v10000_bf16", "distill", 32, 2000, 100, 10000, "path", t_min=1500,
              u_min=60, K=32, rest=True, std=2.0, dtype="bf16"),
        # one hypothesis of one utterance while a user waits
        _case("sample_one_v32000", "sample", 1, 400, 0, 32000, "step", N=1, temperature=0.8,
              top_p=0.9),
        # one step of 64 hypotheses at once
        _case("sample_step_v4096_bf16", "sample", 64, 400, 0, 4096, "step", N=1, top_k=50,
              top_p=0.95, dtype="bf16"),
        # a word at each node of whole alignments (scheduled sampling), the model's own distribution
        _case("sample_path_v1000", "sample", 8, 2000, 100, 1000, "path", t_min=1000, u_min=50),
        # the same over a large vocabulary, without the unlikely words
        _case("sample_path_v10000", "sample", 8, 2000, 100, 10000, "path", t_min=1500, u_min=60,
              top_p=0.9, min_p=0.001),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another case of the same ranges: 1-64 utterances, 1-2000 frames, transcripts of 0-100 labels,
    28-32000 words (half of the vocabularies a multiple of 8), 1-64 words listed per node."""
    while True:
        task = rng.choice(["top", "distill", "distill", "sample", "sample"])
        V = _log(rng, 28, 32000)
        if rng.random() < 0.5:
            V = (V + 7) // 8 * 8
        nodes = rng.choice(["path", "path", "lattice"] if task == "distill"
                           else ["path", "path", "step", "lattice"])
        B = _log(rng, 1, 64 if nodes == "step" else 32)
        T = _log(rng, 1, 2000 if nodes == "path" else 300)
        U = min(_log(rng, 1, 100) - 1, T, 30 if nodes == "lattice" else 100)
        ragged = rng.random() < 0.7
        filters = task == "sample"
        case = _case(None, task, B, T, U, V, nodes,
                     t_min=max(1, int(T * rng.uniform(0.4, 0.9))) if ragged else T,
                     u_min=int(U * rng.uniform(0.2, 0.9)) if ragged else U,
                     N=rng.randint(1, U + 1) if nodes == "step" else 0,
                     K=0 if filters else _log(rng, 1, min(64, V)),
                     rest=task == "distill" and rng.random() < 0.5,
                     temperature=rng.choice([1.0, 1.0, 0.7, 2.0]),
                     top_k=_log(rng, 1, V) if filters and rng.random() < 0.4 else 0,
                     top_p=rng.choice([1.0, 0.5, 0.9, 0.95]) if filters else 1.0,
                     min_p=rng.choice([0.0, 0.0, 0.02, 0.001]) if filters else 0.0,
                     std=rng.choice([1.0, 1.5, 2.0]), dtype=rng.choice(["f32", "f32", "bf16"]),
                     checked=rng.random() < 0.5)
        n = B * _count(case)
        if n * V > (6.4e8 if task == "distill" else 1.6e8) or B * T * V > 6.4e8:
            continue
        return case


def _count(case):
    """Nodes per utterance, those that are none included."""
    if case["nodes"] == "step":
        return case["N"]
    if case["nodes"] == "path":
        return case["T"] + case["U"]
    return case["T"] * (case["U"] + 1)


def _nodes(case, g, dev):
    B, T, U = case["B"], case["T"], case["U"]
    in_lens = torch.randint(case["t_min"], T + 1, (B,), generator=g, device=dev)
    lab_lens = torch.randint(case["u_min"], U + 1, (B,), generator=g, device=dev)
    in_lens[0], lab_lens[0] = T, U
    if case["nodes"] == "step":
        N = case["N"]
        frames = (torch.rand((B, 1), generator=g, device=dev) * in_lens[:, None]).long()
        frames = frames.expand(B, N)
        positions = torch.arange(N, device=dev).expand(B, N)
    elif case["nodes"] == "lattice":
        frames = torch.arange(T, device=dev)[:, None].expand(T, U + 1).reshape(1, -1)
        positions = torch.arange(U + 1, device=dev)[None, :].expand(T, U + 1).reshape(1, -1)
        valid = (frames < in_lens[:, None]) & (positions <= lab_lens[:, None])
        frames = torch.where(valid, frames, -1)
        positions = torch.where(valid, positions, -1)
    else:
        # a random order of the utterance's moves, the last of them a blank's: which ones are labels
        n = torch.arange(T + U, device=dev)[None, :]
        moves = (in_lens + lab_lens)[:, None]
        key = torch.rand((B, T + U), generator=g, device=dev)
        key = torch.where(n < moves - 1, key, 2.0)
        rank = key.argsort(1).argsort(1)
        label = rank < lab_lens[:, None]
        positions = label.cumsum(1) - label.long()
        frames = n - positions
        frames = torch.where(n < moves, frames, -1)
        positions = torch.where(n < moves, positions, -1)
    return frames.int().contiguous(), positions.int().contiguous()


def _raise_words(E, g):
    """On most frames one word, every other time the blank, stands out."""
    B, T, V = E.shape
    word = torch.randint(0, V, (B, T, 1), generator=g, device=E.device)
    word[torch.rand((B, T, 1), generator=g, device=E.device) < 0.5] = 0
    by = 4 + 8 * torch.rand((B, T, 1), generator=g, device=E.device)
    by[torch.rand((B, T, 1), generator=g, device=E.device) < 0.2] = 0
    E.scatter_add_(2, word, by)


def prepare(case, seed):
    dev = torch.device("cuda")
    B, T, U, V = case["B"], case["T"], case["U"], case["V"]
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    rows = case["N"] if case["nodes"] == "step" else U + 1
    E = torch.empty((B, T, V), device=dev).normal_(0.0, case["std"], generator=g)
    P = torch.empty((B, rows, V), device=dev).normal_(0.0, case["std"] / 2, generator=g)
    _raise_words(E, g)
    frames, positions = _nodes(case, g, dev)
    state = {"case": case, "frames": frames, "positions": positions}
    if case["task"] == "distill":
        # the teacher: the student's scores and some disagreement, node by node
        K, N = case["K"], frames.shape[1]
        words = torch.full((B, N, K), -1, device=dev, dtype=torch.int32)
        logits = torch.full((B, N, K), -math.inf, device=dev)
        rest = torch.full((B, N), -math.inf, device=dev)
        for b in range(B):
            z = E[b, frames[b].clamp(min=0).long()]
            z += P[b, positions[b].clamp(min=0).long()]
            z += torch.empty((1, V), device=dev).normal_(0.0, 0.7, generator=g)
            z /= case["temperature"]
            top, at = z.topk(K, dim=1)
            z.scatter_(1, at, -math.inf)
            here = (frames[b] >= 0)[:, None]
            words[b] = torch.where(here, at.int(), -1)
            logits[b] = torch.where(here, top, -math.inf)
            rest[b] = torch.where(here[:, 0], z.logsumexp(1), -math.inf)
            del z
        state.update(words=words, logits=logits, rest=rest if case["rest"] else None)
        state["weights"] = torch.rand((B, N), generator=g, device=dev) / N + 0.5 / N
    if case["task"] == "sample":
        state["uniforms"] = torch.rand(frames.shape, generator=g, device=dev)
    if case["dtype"] == "bf16":
        E, P = E.bfloat16(), P.bfloat16()
    if case["task"] == "distill":
        E.requires_grad_(True)
        P.requires_grad_(True)
    state.update(E=E, P=P)
    if own and case["task"] == "distill":
        from transducer_b200 import NodeDistillationLoss
        state["criterion"] = NodeDistillationLoss(temperature=case["temperature"],
                                                  validate_nodes=case["checked"])
    return state


def run(state):
    case, E, P = state["case"], state["E"], state["P"]
    frames, positions = state["frames"], state["positions"]
    if own:
        if case["task"] == "distill":
            costs = state["criterion"](E, P, frames, positions, state["words"], state["logits"],
                                       state["rest"])
            dE, dP = torch.autograd.grad(costs, (E, P), state["weights"])
            return {"costs": costs.detach(), "dE": dE, "dP": dP}
        import transducer_b200
        if case["task"] == "top":
            words, logits, rest = transducer_b200.top_words(
                E, P, frames, positions, case["K"], temperature=case["temperature"],
                validate_nodes=case["checked"])
            return {"words": words, "logits": logits, "rest": rest}
        words, log_probs = transducer_b200.sample_words(
            E, P, frames, positions, state["uniforms"], temperature=case["temperature"],
            top_k=case["top_k"], top_p=case["top_p"], min_p=case["min_p"],
            validate_nodes=case["checked"])
        return {"words": words, "log_probs": log_probs}
    with torch.no_grad():
        here = (frames >= 0) & (positions >= 0)
        b = torch.arange(E.shape[0], device=E.device)[:, None]
        t, u = frames.clamp(min=0).long(), positions.clamp(min=0).long()
        z = E[b, t].float() + P[b, u].float()
        if case["task"] == "top":
            return _top(case, z, here)
        if case["task"] == "sample":
            return _sample(case, z, here, state["uniforms"])
        costs, g = _distill(case, z, here, state)
        g *= state["weights"][..., None]
        dE = torch.zeros(E.shape, device=E.device).flatten(0, 1)
        dE.index_add_(0, (b * E.shape[1] + t).flatten(), g.flatten(0, 1))
        dP = torch.zeros(P.shape, device=E.device).flatten(0, 1)
        dP.index_add_(0, (b * P.shape[1] + u).flatten(), g.flatten(0, 1))
        return {"costs": costs, "dE": dE.view(E.shape).to(E.dtype),
                "dP": dP.view(P.shape).to(P.dtype)}


def _lse(x):
    m = x.amax(-1, keepdim=True).clamp(min=-3e38)
    return (m + (x - m).exp().sum(-1, keepdim=True).log())[..., 0]


def _top(case, z, here):
    K, tau = case["K"], case["temperature"]
    best, at = z.sort(dim=-1, descending=True, stable=True)
    best = best / tau
    rest = _lse(best[..., K:]) if K < z.shape[-1] else torch.full_like(best[..., 0], -math.inf)
    gone = ~here[..., None]
    return {"words": at[..., :K].int().masked_fill(gone, -1),
            "logits": best[..., :K].masked_fill(gone, -math.inf),
            "rest": rest.masked_fill(~here, -math.inf)}


def _sample(case, z, here, uniforms):
    """In 64 bits: which word a number picks is a comparison with a long sum."""
    best, at = z.sort(dim=-1, descending=True, stable=True)
    w = ((best.double() - best[..., :1].double()) / case["temperature"]).exp()
    del best
    keep = w >= case["min_p"]
    if 0 < case["top_k"] < w.shape[-1]:
        w[..., case["top_k"]:] = 0.0
    if case["top_p"] < 1.0:
        keep &= w.cumsum(-1) - w < case["top_p"] * w.sum(-1, keepdim=True)
    w = torch.zeros_like(w).scatter_(-1, at, w * keep)
    del at, keep
    upto = w.cumsum(-1)
    total = upto[..., -1:]
    word = (upto <= uniforms[..., None].double() * total).sum(-1, keepdim=True)
    log_probs = (w.gather(-1, word) / total).log().float()[..., 0]
    return {"words": word[..., 0].int().masked_fill(~here, -1),
            "log_probs": log_probs.masked_fill(~here, 0.0)}


def _distill(case, z, here, state):
    """Costs, and their gradients with respect to each node's scores."""
    tau, words, rest = case["temperature"], state["words"], state["rest"]
    K = words.shape[-1]
    z = z / tau
    lse = _lse(z)[..., None]
    at = words.clamp(min=0).long()
    bins = state["logits"] if rest is None else torch.cat((state["logits"], rest[..., None]), -1)
    log_q = bins - _lse(bins)[..., None]
    q = log_q.exp()
    log_p = z.gather(-1, at) - lse
    g = (z - lse).exp()
    if rest is not None:
        z.scatter_(-1, at, -math.inf)
        others = _lse(z)[..., None].clamp(min=-3e38)
        log_p = torch.cat((log_p, others - lse), -1)
        g -= q[..., K:] * (z - others).exp()
    costs = torch.where(q > 0, q * (log_q - log_p), 0.0).sum(-1)
    g.scatter_add_(-1, at, -q[..., :K])
    g /= tau
    return costs.masked_fill(~here, 0.0), g.masked_fill_(~here[..., None], 0.0)


def _lengths(case):
    """Expected numbers over the batch: frames with nodes, positions with nodes, nodes."""
    B = case["B"]
    if case["nodes"] == "step":
        return B, B * case["N"], B * case["N"]
    t, u = (case["t_min"] + case["T"]) / 2, (case["u_min"] + case["U"]) / 2
    T, U = case["T"] + (B - 1) * t, case["U"] + (B - 1) * u
    if case["nodes"] == "path":
        return T, U + B, T + U
    return T, U + B, case["T"] * (case["U"] + 1) + (B - 1) * t * (u + 1)


def work(case):
    """The rows that hold nodes read once, the teacher's records and the outputs once (gradients
    whole, padding included).  Per node and word: the sum of the scores, an exponential and its sum,
    a comparison; for distillation a second exponential, the gradient and its two sums."""
    frames, positions, nodes = _lengths(case)
    B, T, U, V, K = case["B"], case["T"], case["U"], case["V"], case["K"]
    size = 2 if case["dtype"] == "bf16" else 4
    slots = B * _count(case)
    nbytes = size * V * (frames + positions) + 8.0 * slots
    if case["task"] == "top":
        return {"bytes": nbytes + slots * (8.0 * K + 4.0), "flops": 4.0 * V * nodes}
    if case["task"] == "sample":
        return {"bytes": nbytes + 12.0 * slots, "flops": 4.0 * V * nodes}
    nbytes += nodes * 8.0 * K + (4.0 * nodes if case["rest"] else 0.0) + 8.0 * slots
    return {"bytes": nbytes + size * V * B * (T + U + 1.0), "flops": 10.0 * V * nodes}


def exact(case, seed):
    """The same from the definitions in 64 bits, one utterance at a time."""
    state = prepare(case, seed)
    E, P, tau, K = state["E"].detach(), state["P"].detach(), case["temperature"], case["K"]
    frames, positions = state["frames"], state["positions"]
    B, N = frames.shape
    first = torch.zeros((B, N), dtype=torch.float64, device=E.device)
    out = {"top": {"words": None, "rest": first - math.inf,
                   "logits": first[..., None].expand(B, N, K) - math.inf},
           "sample": {"words": None, "log_probs": first.clone()},
           "distill": {"costs": first.clone()}}[case["task"]]
    dE, dP = [], []
    for b in range(B):
        e = E[b].double().requires_grad_(case["task"] == "distill")
        p = P[b].double().requires_grad_(case["task"] == "distill")
        n = (frames[b] >= 0).nonzero()[:, 0]
        t, u = frames[b, n].long(), positions[b, n].long()
        if case["task"] == "top":
            z = (e[t] + p[u]) / tau
            top = z.topk(K, dim=1)
            out["logits"][b, n] = top.values
            out["rest"][b, n] = z.scatter(1, top.indices, -math.inf).logsumexp(1)
        elif case["task"] == "sample":
            # (the scores are sums in 32 bits by definition: equal ones are told apart by their place)
            s = E[b, t].float() + P[b, u].float()
            out["log_probs"][b, n] = _exact_sample(case, s, state["uniforms"][b, n])
        else:
            z = (e[t] + p[u]) / tau
            log_p = torch.log_softmax(z, 1)
            at = state["words"][b, n].long()
            bins, at_bins = state["logits"][b, n].double(), log_p.gather(1, at)
            if state["rest"] is not None:
                bins = torch.cat((bins, state["rest"][b, n].double()[:, None]), 1)
                listed_words = torch.zeros_like(z, dtype=torch.bool).scatter(1, at, True)
                others = torch.where(listed_words, -1e300, log_p).logsumexp(1, keepdim=True)
                at_bins = torch.cat((at_bins, others), 1)
            log_q = torch.log_softmax(bins, 1)
            costs = torch.where(log_q > -math.inf, log_q.exp() * (log_q.clamp(min=-1e300) - at_bins),
                                0.0).sum(1)
            out["costs"][b, n] = costs.detach()
            de, dp = torch.autograd.grad(costs, (e, p), state["weights"][b, n].double())
            dE.append(de)
            dP.append(dp)
            del z, log_p
    if case["task"] == "distill":
        out.update(dE=torch.stack(dE), dP=torch.stack(dP))
    return out


def _exact_sample(case, s, uniforms):
    """log-probability of the word that each number picks from its row of `s`."""
    V, k = s.shape[1], case["top_k"]
    w = torch.softmax((s.double() - s.double().amax(1, keepdim=True)) / case["temperature"], 1)
    place = torch.empty_like(s, dtype=torch.int64)
    place.scatter_(1, s.sort(dim=1, descending=True, stable=True).indices,
                   torch.arange(V, device=s.device).expand_as(place).contiguous())
    w = torch.where(place < (k if 0 < k < V else V), w, 0.0)
    kept = w
    if case["top_p"] < 1.0:
        upto = torch.zeros_like(w).scatter_(1, place, w).cumsum(1)
        short = upto < case["top_p"] * upto[:, -1:]
        last = short.sum(1, keepdim=True)   # the place of the word that reaches the share
        kept = torch.where(place <= last, w, 0.0)
    kept = torch.where(w >= case["min_p"] * w.amax(1, keepdim=True), kept, 0.0)
    upto = kept.cumsum(1)
    at = torch.searchsorted(upto, uniforms.double()[:, None] * upto[:, -1:], right=True)
    return (kept.gather(1, at) / upto[:, -1:]).log()[:, 0]
