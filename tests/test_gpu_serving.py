"""GPU: the operators of the 4-bit cache and the sampling of rows together, as a server's loop uses them: prompts of
several sequences as one padded batch, then a token of each per step, on a layer of plain torch products."""
import math

import pytest

import kv4_ref as ref
from test_gpu_kv4 import angles, kv4, noise, torch  # noqa: F401
from test_gpu_sample_rows import definition

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,longest,halves", [(5, 40, False), (18, 60, True)])
def test_prompts_and_steps(torch, kv4, dtype, n, longest, halves):
    from fwb.sampling import sample_rows
    nh, nkv, hd, E, V, steps, page = 16, 4, 64, 256, 1000, 6, 16
    dt = ref.DTYPES[dtype]
    prompts = [longest - i * 17 % (longest - 1) for i in range(n)]
    embed, head = noise(torch, 1, V, E, dtype=dt), noise(torch, 2, nh * hd, V, dtype=dt, sd=0.2)
    wqkv = noise(torch, 3, E, (nh + 2 * nkv) * hd, dtype=dt, sd=1 / math.sqrt(E))
    cos, sin = angles(torch, longest + steps, hd)
    p = ref.Pages(kv4, [0] * n, nkv, hd, page, room=longest + steps)
    gen = torch.Generator(device="cuda").manual_seed(4)
    temperature = torch.tensor([0.0, 0.7, 1.0, 1.3] * n, device="cuda")[:n].contiguous()
    top_k = torch.tensor([0, 40, 0, 5, 0] * n, dtype=torch.int32, device="cuda")[:n].contiguous()
    top_p = torch.tensor([1.0, 0.95, 0.9, 1.0, 0.5, 1.0] * n, device="cuda")[:n].contiguous()
    kv4.check_status()

    def layer(tokens, n_new):
        """The logits of each sequence's last new token."""
        nq = tokens.shape[1]
        x = torch.matmul(embed[tokens], wqkv).view(n, nq, nh + 2 * nkv, hd)
        q, k, v = x[:, :, :nh], x[:, :, nh:nh + nkv], x[:, :, nh + nkv:]
        plan = kv4.Attention(n_seq=n, n_query=nq, n_head=nh, n_head_kv=nkv, head_dim=hd, dtype=dt, page_size=page,
                             n_page=p.n_page, max_pages=p.table.shape[1])
        turned = kv4.append(q, k, v, p.cache, p.table, p.lengths, cos=cos, sin=sin, halves=halves, n_new=n_new)
        out, lse = plan(turned, p.cache, p.table, p.lengths, n_new=n_new)
        kk, vv = kv4.read(p.cache, p.table, torch.zeros_like(p.lengths), longest + steps, head_dim=hd, dtype=torch.float32, lengths=p.lengths)
        ref.check_attention(out, lse, turned, kk, vv, p.lengths.tolist(), n_new.tolist())
        for s in range(n):                                         # what the last append left in the cache
            fresh, end = int(n_new[s]), int(p.lengths[s])
            want = ref.held(ref.turned(k[s, :fresh], cos[end - fresh:end], sin[end - fresh:end], halves))
            assert torch.equal(kk[s, end - fresh:end].double(), want)
        return torch.matmul(out[torch.arange(n, device="cuda"), n_new.long() - 1].flatten(1), head)

    tokens = torch.randint(0, V, (n, longest), device="cuda", generator=gen)
    n_new = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    p.lengths.copy_(n_new)
    for _ in range(steps):
        logits = layer(tokens, n_new)
        u = torch.rand(n, device="cuda", generator=gen)
        token, logprob = sample_rows(logits, u, temperature=temperature, top_k=top_k, top_p=top_p)
        for s in range(n):
            want, lp, clear, near = definition(torch, logits[s], float(u[s]), float(temperature[s]), int(top_k[s]), float(top_p[s]), 0.0)
            assert int(token[s]) == want or (clear < 2.0 ** -20 and int(token[s]) in near)
            assert clear < 2.0 ** -20 or abs(float(logprob[s]) - lp) <= 2.0 ** -20 + abs(lp) * 2.0 ** -22
        tokens = token.long()[:, None]
        n_new = torch.ones(n, dtype=torch.int32, device="cuda")
        p.lengths.add_(1)
    kv4.check_status()
