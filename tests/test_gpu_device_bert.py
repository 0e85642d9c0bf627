"""DeviceBert's own buffers: which stream they belong to, and what a change of shape or of attention leaves of them."""
import numpy as np
import pytest

from aikit_amd import enchip
from aikit_amd.bert_dev import DeviceBert
from test_gpu_attention_block import layers_of

pytestmark = pytest.mark.gpu

D, H, I, HD = 128, 4, 256, 32
SHAPES = [(4, 64), (2, 96), (4, 63)]  # the third's buffers fit where the first's were


def say(msg):
    print(f"[case] {msg}", flush=True)


@pytest.fixture
def model(ctx):
    m = DeviceBert(ctx, layers_of(np.random.default_rng(5), 2, D, 3 * D, I, HD, False, False), D, H, I)
    yield m
    m.close()


def hidden(torch, S, L):
    return torch.from_numpy(np.random.default_rng(S * L).standard_normal((S * L, D)).astype(np.float32)).cuda()


def sleep(torch, stream=None):  # about 50 ms of the shader clock
    with torch.cuda.stream(stream or torch.cuda.current_stream()):
        torch.cuda._sleep(100_000_000)


def alone(torch, model, stream=0):
    out = []
    for S, L in SHAPES:
        h, p = hidden(torch, S, L), torch.zeros((S, D), device="cuda")
        torch.cuda.synchronize()
        model.embed(h, S, L, p, stream)
        torch.cuda.synchronize()
        out.append((h.cpu().numpy(), p.cpu().numpy()))
    return out


def test_the_contexts_stream(ctx):
    import torch

    s = ctx.stream()
    assert s and s == ctx.stream()
    x = torch.full((4, 8), 2.0, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.ExternalStream(s)):
        x.mul_(3.0)
        x.add_(1.0)
    torch.cuda.synchronize()
    assert (x == 7.0).all()
    assert enchip.load().enchip_stream(ctx.handle, None) == enchip.ERR_ARG


@pytest.mark.parametrize("own", [True, False])
def test_shapes_queued_behind_each_other(ctx, model, own):
    import torch

    say(f"three shapes queued behind each other, on the context's stream: {own}")
    want = alone(torch, model)
    for busy in (True, False):  # torch's stream far behind the layers' stream, or far ahead of it
        st = torch.cuda.Stream()
        sp = ctx.stream() if own else st.cuda_stream
        model._bufs = {}
        hs = [hidden(torch, *k) for k in SHAPES]
        ps = [torch.zeros((S, D), device="cuda") for S, _ in SHAPES]
        torch.cuda.synchronize()
        sleep(torch, None if busy else torch.cuda.ExternalStream(sp))
        for (S, L), h, p in zip(SHAPES, hs, ps):
            model.embed(h, S, L, p, 0 if own else sp)
        # tensors of the caller's, of the dropped buffers' sizes, while the first shapes may still be queued
        mine = [torch.full((S * L, w), 7.0, device="cuda") for S, L in SHAPES for w in (3 * D, D, I, D, D)]
        torch.cuda.synchronize()
        for (h, p), a, b in zip(want, hs, ps):
            assert np.array_equal(a.cpu().numpy(), h) and np.array_equal(b.cpu().numpy(), p), busy
        for t in mine:
            assert (t == 7.0).all(), busy


def test_nothing_of_torchs_stream_lands_between_the_layers(ctx, model):
    # everything torch has queued lands after the attention and before the linear that reads its output
    import torch

    say("a new shape behind a busy torch stream")
    want = alone(torch, model)
    for i, (S, L) in enumerate(SHAPES):
        h, p = hidden(torch, S, L), torch.zeros((S, D), device="cuda")
        torch.cuda.synchronize()
        model._bufs = {}
        sleep(torch)
        model.mark = lambda label: torch.cuda.synchronize() if label.startswith("o") else None
        try:
            model.embed(h, S, L, p)
            torch.cuda.synchronize()
        finally:
            model.mark = None
        assert np.array_equal(h.cpu().numpy(), want[i][0]) and np.array_equal(p.cpu().numpy(), want[i][1])


@pytest.mark.parametrize("L", [70, 1])
def test_buffers_of_a_shape_stay_where_a_graph_has_them(ctx, L):
    # heads without a fused attention keep scores, which spans do not need: the shape's other buffers stay
    import torch

    S = 2
    g = np.random.default_rng(8)
    m = DeviceBert(ctx, layers_of(g, 1, D, 3 * D, I, HD, False, False), D, H, I, fused=False)
    say(f"a captured forward over spans, then one without them, {S} x {L}")
    try:
        st = torch.cuda.Stream()
        x = hidden(torch, S, L)
        spans = torch.tensor([[0, L], [L, 2 * L]], dtype=torch.int32, device="cuda")
        h, p, q = x.clone(), torch.zeros((S, D), device="cuda"), torch.zeros((S, D), device="cuda")
        torch.cuda.synchronize()
        m.embed(h, S, L, p, st.cuda_stream, spans=spans)
        torch.cuda.synchronize()
        want = p.cpu().numpy()
        held = {k: (t, t.data_ptr()) for k, t in m._bufs[(S, L)].items() if k != "scores"}
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            m.embed(h, S, L, p, st.cuda_stream, spans=spans)
        for _ in range(3):
            h.copy_(x)
            torch.cuda.synchronize()
            m.embed(h, S, L, q, st.cuda_stream)  # its scores in a buffer of its own
            torch.cuda.synchronize()
            assert all(m._bufs[(S, L)][k] is t and t.data_ptr() == at for k, (t, at) in held.items())
            # unit vectors whose cosine is at least the encoders' bar of 0.9999
            assert (np.linalg.norm(q.cpu().numpy() - want, axis=1) <= (2e-4) ** 0.5).all()
            h.copy_(x)
            p.zero_()
            torch.cuda.synchronize()
            gr.replay()
            torch.cuda.synchronize()
            assert np.array_equal(p.cpu().numpy(), want)
        del gr
    finally:
        m.close()


def test_more_spans_than_one_call_pools(ctx, model):
    import torch

    n, L = 70000, 66000
    say(f"embed {n} spans, most of them empty")
    g = np.random.default_rng(12)
    size = np.zeros(n, np.int64)
    some = np.sort(g.choice(n, 600, replace=False))
    some[-1] = n - 1
    size[some] = g.integers(1, 100, 600)
    end = np.cumsum(size)
    assert end[-1] <= L
    spans = np.stack([end - size, end], axis=1).astype(np.int32)
    x = torch.from_numpy(g.standard_normal((L, D)).astype(np.float32)).cuda()
    out = []
    for keep in (np.arange(n), some):
        h, p = x.clone(), torch.full((len(keep) + 1, D), 5.0, device="cuda")
        sp = torch.from_numpy(spans[keep]).cuda()
        torch.cuda.synchronize()
        model.embed(h, 1, L, p, spans=sp)
        torch.cuda.synchronize()
        out.append(p.cpu().numpy())
    many, few = out
    empty = np.ones(n, bool)
    empty[some] = False
    assert (many[-1] == 5.0).all() and (many[:n][empty] == 0).all()
    # the order of the attention's sums goes by L / n: codes on a rounding border, the encoders' bar of 0.9999
    assert (np.linalg.norm(many[some] - few[:-1], axis=1) <= (2e-4) ** 0.5).all()


def test_a_captured_shape_keeps_its_buffers(ctx, model):
    # a graph's replay writes where its shape's buffers were: they are nobody else's after other shapes have run
    import torch

    st = torch.cuda.Stream()
    S, L = SHAPES[0]
    x, h = hidden(torch, S, L), hidden(torch, S, L)
    p = torch.zeros((S, D), device="cuda")
    torch.cuda.synchronize()
    model.embed(h, S, L, p, st.cuda_stream)
    torch.cuda.synchronize()
    want = p.cpu().numpy()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=st):
        model.embed(h, S, L, p, st.cuda_stream)
    say("a captured shape, other shapes, tensors of its buffers' sizes, its replays")
    for rep in range(3):
        for S2, L2 in SHAPES[1:] + [(1, 17)]:
            h2, p2 = hidden(torch, S2, L2), torch.zeros((S2, D), device="cuda")
            torch.cuda.synchronize()
            model.embed(h2, S2, L2, p2, st.cuda_stream)
        with torch.cuda.stream(st):
            mine = [torch.full((S * L, w), 7.0, device="cuda") for w in (3 * D, D, I, D, D) for _ in range(3)]
            h.copy_(x)
            p.zero_()
        torch.cuda.synchronize()
        gr.replay()
        torch.cuda.synchronize()
        assert np.array_equal(p.cpu().numpy(), want), rep
        for t in mine:
            assert (t == 7.0).all(), rep
    del gr
