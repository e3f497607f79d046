"""64-bit causal attention with a window and sinks, from its definition (for test_window_gpu.py and the paged cache's tests)."""
import torch


def visible(nq, nk, window, sinks, device=None):
    """(nq, nk) truth values: key j is seen by the query at position p = nk - nq + i if j <= p, and j > p - window or j < sinks."""
    pos = torch.arange(nq, device=device)[:, None] + nk - nq
    key = torch.arange(nk, device=device)[None]
    return (key <= pos) & ((key > pos - window) | (key < sinks))


def window_reference(q, k, v, ql, kl, window, sinks, scale):
    """o (total_q, H, D) and lse (H, total_q); differentiable. Queries without keys: 0 and -inf."""
    group = q.size(1) // k.size(1)
    outs, lses, q0, k0 = [], [], 0, 0
    for nq, nk in zip(ql, kl):
        qs = q[q0:q0 + nq].transpose(0, 1)
        ks, vs = (t[k0:k0 + nk].repeat_interleave(group, 1).transpose(0, 1) for t in (k, v))
        seen = visible(nq, nk, window, sinks, q.device)
        s = torch.where(seen, qs @ ks.transpose(1, 2) * scale, float("-inf"))
        top = s.detach().amax(-1, keepdim=True).clamp_min(-1e300) if nk else s.new_zeros(q.size(1), nq, 1)
        e = torch.where(seen, torch.exp(s - top), 0.0)
        total = e.sum(-1, keepdim=True)
        outs.append(((e / torch.where(total == 0, 1.0, total)) @ vs).transpose(0, 1))
        lses.append((top + torch.log(total))[..., 0])
        q0, k0 = q0 + nq, k0 + nk
    return torch.cat(outs), torch.cat(lses, 1)
