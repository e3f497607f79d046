"""64-bit attention over packed sequences, from its definition (for test_packed_gpu.py, test_paged_gpu.py)."""
import torch


def packed_reference(q, k, v, ql, kl, causal, scale):
    """o (total_q, H, D) and lse (H, total_q); differentiable. Queries without keys: 0 and -inf."""
    group = q.size(1) // k.size(1)
    outs, lses, q0, k0 = [], [], 0, 0
    for nq, nk in zip(ql, kl):
        qs = q[q0:q0 + nq].transpose(0, 1)
        ks, vs = (t[k0:k0 + nk].repeat_interleave(group, 1).transpose(0, 1) for t in (k, v))
        seen = torch.ones(nq, nk, dtype=torch.bool, device=q.device)
        if causal:
            seen = torch.arange(nk, device=q.device)[None] <= torch.arange(nq, device=q.device)[:, None] + nk - nq
        s = torch.where(seen, qs @ ks.transpose(1, 2) * scale, float("-inf"))
        top = s.detach().amax(-1, keepdim=True).clamp_min(-1e300) if nk else s.new_zeros(q.size(1), nq, 1)
        e = torch.where(seen, torch.exp(s - top), 0.0)
        total = e.sum(-1, keepdim=True)
        outs.append(((e / torch.where(total == 0, 1.0, total)) @ vs).transpose(0, 1))
        lses.append((top + torch.log(total))[..., 0])
        q0, k0 = q0 + nq, k0 + nk
    return torch.cat(outs), torch.cat(lses, 1)
