"""GPU: CUDA graphs captured from one plan of fwb.beam are independent of each
other and of the plan's other calls."""
import pytest

from test_gpu_beam import attn_case, beam, torch  # noqa: F401

pytestmark = pytest.mark.gpu


def side_by_side(torch, plain, calls, outs, wants):
    """One graph for each call, all captured on torch's own capture stream, replayed on streams of their own beside the
    uncaptured call `plain`, which has the first of the outputs."""
    graphs = []
    for call in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        for _ in range(5):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
            plain()
        torch.cuda.synchronize()
        for o, want in zip(outs, wants):
            assert all(torch.equal(a, b) for a, b in zip(o, want))


def test_attention_graphs_side_by_side(torch, beam):
    c = attn_case(torch, "f16", 1, 6, 1, 8, 2, 128, 6000, 30)
    plan = beam.PrefixAttention(n_group=1, n_beam=6, n_head=8, n_head_kv=2, head_dim=128, dtype=torch.float16,
                                prefix_cap=6000, suffix_cap=30)
    kv = [c[k] for k in ("pk", "pv", "sk", "sv")]
    qs = [c["q"], c["q"].flip(0).contiguous(), c["q"] * 0.5]
    wants = [plan(q, *kv, slots=c["slots"]) for q in qs]
    outs = [tuple(torch.empty_like(t) for t in w) for w in wants]
    eager = tuple(torch.empty_like(t) for t in wants[0])
    calls = [lambda q=q, o=o: plan(q, *kv, slots=c["slots"], out=o[0], lse=o[1]) for q, o in zip(qs, outs)]
    side_by_side(torch, lambda: plan(qs[0], *kv, slots=c["slots"], out=eager[0], lse=eager[1]), calls, [eager] + outs,
                 wants[:1] + wants)


def test_select_graphs_side_by_side(torch, beam):
    gen = torch.Generator(device="cuda").manual_seed(1)
    plan = beam.BeamSelect(n_group=2, n_beam=4, n_vocab=32000, n_select=8)
    xs = [torch.randn(2, 4, 32000, device="cuda", generator=gen) for _ in range(3)]
    scores = torch.zeros(2, 4, device="cuda")
    wants = [plan(x, scores) for x in xs]
    outs = [tuple(torch.empty_like(t) for t in w) for w in wants]
    eager = tuple(torch.empty_like(t) for t in wants[0])
    calls = [lambda x=x, o=o: plan(x, scores, *o) for x, o in zip(xs, outs)]
    side_by_side(torch, lambda: plan(xs[0], scores, *eager), calls, [eager] + outs, wants[:1] + wants)


def test_a_graph_outlives_its_plan(torch, beam):
    c = attn_case(torch, "bf16", 1, 6, 1, 8, 2, 128, 3000, 30)
    plan = beam.PrefixAttention(n_group=1, n_beam=6, n_head=8, n_head_kv=2, head_dim=128, dtype=torch.bfloat16,
                                prefix_cap=3000, suffix_cap=30)
    args = [c[k] for k in ("q", "pk", "pv", "sk", "sv")]
    want, lse = plan(*args, slots=c["slots"])
    out = torch.empty_like(want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan(*args, slots=c["slots"], out=out, lse=lse)
    size = plan.workspace_bytes
    del plan
    for _ in range(20):
        other = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(4)]
        out.zero_()
        g.replay()
        assert torch.equal(out, want) and all(bool((o == 255).all()) for o in other)
