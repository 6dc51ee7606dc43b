"""The node operators from their definitions, in 64 bits on the CPU: what the kernels are held to.
The scores are the 32-bit sums that the operators are defined on."""
import torch


def scores(E, P, frames, positions):
    """z [B, N, V] float32 and which nodes exist; rows of zeros where there is none."""
    E, P, frames, positions = (x.detach().cpu() for x in (E, P, frames, positions))
    here = (frames >= 0) & (frames < E.shape[1]) & (positions >= 0) & (positions < P.shape[1])
    b = torch.arange(E.shape[0])[:, None].expand(frames.shape)
    z = torch.zeros(*frames.shape, E.shape[2])
    z[here] = E[b[here], frames[here].long()].float() + P[b[here], positions[here].long()].float()
    return z, here


def order(z):
    """Places of the words, the greater score first, of equal ones the lower word."""
    return torch.sort(z, dim=-1, descending=True, stable=True).indices


def lse(x):
    m = x.amax(-1, keepdim=True).clamp(min=-1e300)
    return (m + (x - m).exp().sum(-1, keepdim=True).log())[..., 0]


def top_words(z, here, k, temperature=1.0):
    at = order(z)
    x = z.double() / temperature
    logits = x.gather(-1, at[..., :k])
    others = x.scatter(-1, at[..., :k], -torch.inf)
    return (at[..., :k].int().masked_fill(~here[..., None], -1),
            logits.masked_fill(~here[..., None], -torch.inf),
            lse(others).masked_fill(~here, -torch.inf))


def sample_words(z, here, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    V = z.shape[-1]
    m = z.amax(-1, keepdim=True).double()
    if temperature == 0.0:
        words = order(z)[..., 0]
        log_probs = torch.zeros(z.shape[:-1], dtype=torch.float64)
    else:
        w = ((z.double() - m) / temperature).exp()
        at = order(z)
        ws = w.gather(-1, at)
        stays = torch.ones_like(ws, dtype=torch.bool)
        if 0 < top_k < V:
            stays[..., top_k:] = False
        if top_p < 1.0:
            left = ws * stays
            stays &= left.cumsum(-1) - left < top_p * left.sum(-1, keepdim=True)
        stays &= ws >= min_p
        w = torch.zeros_like(w).scatter(-1, at, ws * stays)
        upto = w.cumsum(-1)
        # (outside [0, 1): the nearest 32-bit number in it)
        u = uniforms.cpu().double().nan_to_num(nan=1.0).clamp(0.0, 1.0 - 2.0 ** -24)[..., None]
        words = (upto <= u * upto[..., -1:]).sum(-1).clamp(max=V - 1)
        log_probs = (w.gather(-1, words[..., None]) / upto[..., -1:]).log()[..., 0]
    words = words.int()
    masked = m[..., 0] == -torch.inf
    broken = z.isnan().any(-1) | (z == torch.inf).any(-1)
    words = words.masked_fill(masked | broken | ~here, -1)
    log_probs = log_probs.masked_fill(masked, -torch.inf).masked_fill(broken, torch.nan)
    return words, log_probs.masked_fill(~here, 0.0)


def distill(z, here, words, logits, rest=None, temperature=1.0):
    """costs [B, N], their gradients with respect to the scores [B, N, V], and a bound per entry, in
    units of the rounding of 32-bit numbers, on what the kernel's roundings add up to (see below)."""
    B, N, V = z.shape
    words, logits = words.cpu(), logits.cpu().double()
    K = words.shape[-1]
    # (relative to the row's greatest score: next to -3e38 a logarithm would be lost, in 64 bits too)
    m = z.amax(-1, keepdim=True)
    x = (z.double() - torch.where(m > -torch.inf, m, 0.0).double()) / temperature
    there = (words >= 0) & (words < V) & here[..., None]
    l = logits.masked_fill(~there, -torch.inf)
    if rest is not None:
        l = torch.cat((l, rest.cpu().double()[..., None]), -1)
    full = (l > -torch.inf).any(-1) & here
    # (the teacher's too relative to its greatest: shares that add up to 1, at -3e38 as elsewhere)
    l = l - torch.where(l.amax(-1, keepdim=True) > -torch.inf, l.amax(-1, keepdim=True), 0.0)
    q_bins = torch.where(full[..., None], (l - lse(l)[..., None]).exp(), 0.0)
    at = words.clamp(0, V - 1).long()
    q = torch.zeros_like(x).scatter_add_(-1, at, torch.where(there, q_bins[..., :K], 0.0))
    listed = torch.zeros_like(x).scatter_add_(-1, at, there.double()) > 0
    some = (x > -torch.inf).any(-1, keepdim=True)
    L = lse(x)[..., None]
    log_p = torch.where(some & (x > -torch.inf), x - torch.where(some, L, 0.0), -torch.inf)
    costs = torch.where(q > 0, q * (q.clamp(min=1e-300).log() - log_p), 0.0).sum(-1)
    size = torch.where(q > 0, q * (q.clamp(min=1e-300).log().abs() + log_p.abs()), 0.0).sum(-1)
    p = log_p.exp() * full[..., None]
    g = p - q
    grad_size = p + q
    if rest is not None:
        r = q_bins[..., K:]
        xo = x.masked_fill(listed, -torch.inf)
        R = lse(xo)[..., None]
        some_other = (xo > -torch.inf).any(-1, keepdim=True)
        log_rho = torch.where(some_other, R - torch.where(some, L, 0.0), -torch.inf)
        costs += torch.where(r > 0, r * (r.clamp(min=1e-300).log() - log_rho), 0.0)[..., 0]
        size += torch.where(r > 0, r * (r.clamp(min=1e-300).log().abs() + log_rho.abs()), 0.0)[..., 0]
        e = torch.where(some_other, (xo - torch.where(some_other, R, 0.0)).exp(), 0.0)
        g = g - r * e
        grad_size = grad_size + r * e
    # Rounding: a score's distance from the row's maximum is rounded, scaled (the scale is rounded
    # too) and joined with the log-normaliser: 4 roundings of |x - m|; exponentials, sums over a
    # thread's words and over the group, the teacher's sum over its K words: below 64 + K.
    span = torch.where(x > -torch.inf, (x.amax(-1, keepdim=True).clamp(min=-1e300) - x), 0.0)
    span = span.masked_fill(log_p < -80.0, 0.0)   # (such a word's share is 0 in 32 bits or nearly so)
    units = 64.0 + K + 4.0 * span
    costs = torch.where(here, costs, 0.0)
    top_span = torch.where(q > 0, q * span, 0.0).sum(-1)
    cost_bound = (64.0 + K) * size + 4.0 * top_span + 64.0
    g = torch.where(full[..., None], g, 0.0) / temperature
    return costs, g, cost_bound, units * grad_size / temperature


def spread(E, P, frames, positions, here, per_node):
    """Sums of per_node [B, N, V] over the nodes of each frame and of each position."""
    B, T, V = E.shape
    U = P.shape[1]
    de = torch.zeros(B, T, V, dtype=torch.float64)
    dp = torch.zeros(B, U, V, dtype=torch.float64)
    for b in range(B):
        n = here[b].nonzero()[:, 0]
        de[b].index_add_(0, frames[b].cpu()[n].long(), per_node[b, n])
        dp[b].index_add_(0, positions[b].cpu()[n].long(), per_node[b, n])
    return de, dp
