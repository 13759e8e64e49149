"""Edges of the prompt and logits operators: a step of all three captured and replayed, two
contexts at once, offsets past 32 bits, heads of every width."""
import numpy as np
import pytest

import paged_ref as ref
import prompt_ref
from test_gpu_prompt import make, run, tolerance

pytestmark = pytest.mark.gpu
TYPES = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}


class Step:
    """Projection rows in, a chosen token per request out, on torch tensors: head norms and
    rotation with append, prompt attention, a head of its own, penalties and a mask."""

    def __init__(self, torch, ctx, dtype, rows, past=None, H=8, K=2, D=64, page=16, vocab=1000, seed=0):
        from chat_wgpu_b200.kernels import logits, prompt, rope
        self.torch, self.dtype, self.D, self.H, self.K = torch, dtype, D, H, K
        dt = getattr(torch, TYPES[dtype])
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        i = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
        n, T = len(rows), sum(rows)
        self.n, self.T, self.rows_of, self.page = n, T, rows, page
        self.starts = np.concatenate([[0], np.cumsum(rows)])
        self.w = (H + 2 * K) * D
        self.proj = torch.zeros(T, self.w, dtype=dt, device="cuda")
        self.head = torch.randn(H * D, vocab, generator=self.g, device="cuda") / (H * D) ** 0.5
        self.qn, self.kn = (1 + 0.1 * torch.randn(D, generator=self.g, device="cuda") for _ in range(2))
        self.q, self.k = (torch.empty(T, x * D, dtype=dt, device="cuda") for x in (H, K))
        self.pages = -(-T // page) + 1
        self.kc, self.vc = (torch.zeros(self.pages, K, page, D, dtype=dt, device="cuda") for _ in range(2))
        self.pos = np.concatenate([np.arange(r) for r in rows])
        self.slots = np.random.default_rng(seed).permutation(self.pages * page)[:T]
        self.o = torch.empty(T, H * D, dtype=dt, device="cuda")
        self.last = torch.tensor(self.starts[1:] - 1, device="cuda")
        self.logits, self.out = (torch.empty(n, vocab, device="cuda") for _ in range(2))
        self.best = i([0] * n)
        self.tokens = [[3, 4, 5, 3] * (r % 5 + 1) for r in range(n)]
        at = np.concatenate([[0], np.cumsum([len(t) for t in self.tokens])])
        allow = np.random.default_rng(seed + 1).random((1, vocab)) < 0.5
        self.allow = allow
        bits = np.zeros((1, -(-vocab // 32) * 32), np.uint8)
        bits[:, :vocab] = allow
        words = torch.tensor(np.packbits(bits, axis=1, bitorder="little").view(np.int32), device="cuda")
        w = ctx.wrap
        q, k, v = self.proj.split([H * D, K * D, K * D], dim=1)
        self.keep = (q, k, v, words)
        self.norm = rope.NormRope(
            ctx, plan=rope.rope_plan(ctx, D, 1e4), positions=w(i(self.pos.tolist())), dtype=dtype, n_tokens=T,
            head_dim=D, eps=1e-6, n_heads=H, n_kv=K, q=w(q), q_stride=self.w, q_norm=w(self.qn), q_out=w(self.q),
            k=w(k), k_stride=self.w, k_norm=w(self.kn), k_out=w(self.k), v=w(v), v_stride=self.w,
            slots=w(i(self.slots.tolist())), k_cache=w(self.kc), v_cache=w(self.vc), page_size=page,
            n_pages=self.pages)
        self.attend = prompt.PromptAttention(
            ctx, q=w(self.q), k=w(self.k), v=w(v), v_stride=self.w, starts=w(i(self.starts.tolist())), out=w(self.o),
            dtype=dtype, n_req=n, n_rows=T, n_heads=H, n_kv=K, head_dim=D)
        self.adjust = logits.AdjustLogits(
            ctx, logits=w(self.logits), out=w(self.out), dtype="f32", n_rows=n, vocab=vocab,
            penalties=w(torch.tensor([[1.2, 0.1, 0.2]] * n, device="cuda")), tokens=w(i(sum(self.tokens, []))),
            starts=w(i(at.tolist())), n_tokens=int(at[-1]), masks=w(words), n_masks=1, mask_rows=w(i([0] * n)),
            best=w(self.best))

    def fill(self, seed):
        g = self.torch.Generator(device="cuda").manual_seed(seed)
        self.proj.copy_(self.torch.randn(self.proj.shape, generator=g, device="cuda"))

    def __call__(self):
        self.norm()
        self.attend()
        self.torch.mm(self.o[self.last].float(), self.head, out=self.logits)
        self.adjust()

    def check(self):
        """Every stage against the 64-bit form of what went into it."""
        H, K, D, T = self.H, self.K, self.D, self.T
        val = lambda t: t.double().cpu().numpy()  # noqa: E731
        p = val(self.proj)
        f, amp = ref.rates(D, 1e4)
        u = 0 if self.dtype == "f32" else ref.UNIT[self.dtype]
        for got, x, heads, wt in ((self.q, p[:, :H * D], H, self.qn), (self.k, p[:, H * D:(H + K) * D], K, self.kn)):
            want = prompt_ref.norm_rotate(x.reshape(T, heads, D), val(wt), False, 1e-6, self.pos, f, amp, "half")
            # norm and rotation below 2^-18 of the head's largest pair, one rounding
            tol = 2.0 ** -18 * 2 * np.abs(want).max(-1, keepdims=True) + u * np.abs(want)
            assert (np.abs(val(got).reshape(want.shape) - want) <= tol).all()
        s = self.slots
        assert np.array_equal(val(self.vc)[s // self.page, :, s % self.page].reshape(T, -1), p[:, (H + K) * D:])
        assert np.array_equal(val(self.kc)[s // self.page, :, s % self.page].reshape(T, -1), val(self.k))
        want, big_s, big_v = prompt_ref.attention(
            val(self.q).reshape(T, H, D), val(self.k).reshape(T, K, D), p[:, (H + K) * D:].reshape(T, K, D),
            self.starts, self.starts, 0, 0.0, D ** -0.5, np.zeros((T, H, D)))
        assert np.abs(val(self.o).reshape(T, H, D) - want).max() <= tolerance(self.dtype, big_s, big_v, T)
        want, best = prompt_ref.adjust(self.logits.cpu().numpy(), "f32", [(1.2, 0.1, 0.2)] * self.n, self.tokens, None,
                                       None, self.allow, [0] * self.n)
        assert np.array_equal(self.out.double().cpu().numpy(), want)
        assert np.array_equal(self.best.cpu().numpy(), best)


@pytest.mark.parametrize("dtype,rows", [("bf16", [130, 1, 40]), ("f16", [900, 7]), ("f32", [300, 1, 77])])
def test_step_captured_and_replayed(dtype, rows):
    """The three operators as a step uses them, run, captured and replayed on other values, on
    a stream of the caller's; another call of other sizes between the replays."""
    torch = pytest.importorskip("torch")
    from chat_wgpu_b200 import GpuContext
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        c = GpuContext(0, stream=side.cuda_stream)
        step, other = (Step(torch, c, dtype, r) for r in (rows, [5, 600]))
        step.fill(1)
        step()
        side.synchronize()
        step.check()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        for seed in (2, 3):
            step.fill(seed)
            for t in (step.q, step.k, step.o, step.out, step.kc, step.vc):
                t.zero_()
            graph.replay()
            side.synchronize()
            step.check()
            other.fill(seed)
            other()
            side.synchronize()
            other.check()
        c.sync()
        del graph
        c.close()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_two_contexts_at_once(dtype):
    """Calls in flight on two streams, with items that are cut: each context its own scratch."""
    torch = pytest.importorskip("torch")
    from chat_wgpu_b200 import GpuContext
    from chat_wgpu_b200.kernels import prompt
    dt, H, K, D, keys = getattr(torch, TYPES[dtype]), 8, 2, 128, 3000
    g = torch.Generator(device="cuda").manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dt)  # noqa: E731
    i = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    calls, keep = [], []
    for rows in (5, 9):
        st = torch.cuda.Stream()
        c = GpuContext(0, stream=st.cuda_stream)
        t = dict(q=rnd(rows, H * D), k=rnd(keys, K * D), v=rnd(keys, K * D), out=torch.empty(rows, H * D, dtype=dt, device="cuda"),
                 starts=i([0, rows]), key_starts=i([0, keys]))
        torch.cuda.synchronize()
        calls.append(prompt.PromptAttention(c, **{k: c.wrap(x) for k, x in t.items()}, dtype=dtype, n_req=1, n_rows=rows,
                                            n_keys=keys, n_heads=H, n_kv=K, head_dim=D))
        keep.append((c, t, st))
    for _ in range(20):
        for call in calls:
            call()
    for c, t, st in keep:
        c.sync()
        val = lambda x: x.double().cpu().numpy()  # noqa: E731
        rows = t["q"].shape[0]
        want, s, v = prompt_ref.attention(val(t["q"]).reshape(rows, H, D), val(t["k"]).reshape(keys, K, D),
                                          val(t["v"]).reshape(keys, K, D), [0, rows], [0, keys], 0, 0.0, D ** -0.5,
                                          np.zeros((rows, H, D)))
        assert np.abs(val(t["out"]).reshape(rows, H, D) - want).max() <= tolerance(dtype, s, v, keys)
        c.close()


@pytest.mark.parametrize("rows", [9, 200])
def test_every_head_dim(ctx, rows):
    """Head dims of every instance and between them, of one block and of several."""
    for D in [*range(8, 257, 24), 1, 6, 63, 65, 127, 129, 256]:
        for dtype in ("f32", "bf16" if D % 16 else "f16"):
            c = make(np.random.default_rng(D), [rows, 3], [rows + 5, 3], dtype, 4, 2, D)
            got = run(ctx, c, dtype)
            want, s, v = prompt_ref.attention(c["q"], c["k"], c["v"], c["starts"], c["ks"], 0, 0.0, D ** -0.5, c["q"])
            assert np.abs(got - want).max() <= tolerance(dtype, s, v, rows + 5), (D, dtype)
            ctx.sync()


@pytest.mark.parametrize("dtype,rows", [("bf16", 300), ("f32", 300), ("bf16", 3)])
def test_far_rows(dtype, rows):
    """Strides that put rows past 32-bit element offsets give what rows side by side give."""
    torch = pytest.importorskip("torch")
    from chat_wgpu_b200 import GpuContext
    from chat_wgpu_b200.kernels import prompt, rope
    dt, H, K, D, T, wide = getattr(torch, TYPES[dtype]), 4, 2, 64, 300, 1 << 23
    g = torch.Generator(device="cuda").manual_seed(2)
    far = torch.empty(T, wide, dtype=dt, device="cuda")  # 2.5e9 elements
    near = torch.randn(T, (H + 2 * K) * D, generator=g, device="cuda").to(dt)
    far[:, :near.shape[1]] = near
    i = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    c = GpuContext(0, stream=torch.cuda.current_stream().cuda_stream)
    outs = []
    for x in (near, far):
        q, k, v = x[:, :H * D], x[:, H * D:(H + K) * D], x[:, (H + K) * D:(H + 2 * K) * D]
        o = torch.empty(rows, H * D, dtype=dt, device="cuda")
        prompt.PromptAttention(c, q=c.wrap(q[T - rows:]), k=c.wrap(k), v=c.wrap(v), starts=c.wrap(i([0, rows])),
                               key_starts=c.wrap(i([0, T])), out=c.wrap(o), dtype=dtype, n_req=1, n_rows=rows, n_keys=T,
                               n_heads=H, n_kv=K, head_dim=D, q_stride=x.stride(0), k_stride=x.stride(0),
                               v_stride=x.stride(0))()
        ko = torch.empty(T, K * D, dtype=dt, device="cuda")
        qo = torch.empty(T, H * D, dtype=dt, device="cuda")
        rope.NormRope(c, plan=rope.rope_plan(c, D, 1e4), positions=c.wrap(i(list(range(T)))), dtype=dtype, n_tokens=T,
                      head_dim=D, eps=1e-6, n_heads=H, n_kv=K, q=c.wrap(q), q_stride=x.stride(0), q_out=c.wrap(qo),
                      k=c.wrap(k), k_stride=x.stride(0), k_out=c.wrap(ko),
                      q_norm=c.wrap(torch.ones(D, device="cuda")))()
        c.sync()
        outs.append((o, qo, ko))
    for a, b in zip(*outs):
        assert bool(a.isfinite().all()) and torch.equal(a, b)
    c.close()
    del far
    torch.cuda.empty_cache()


def test_far_logits():
    """Rows whose elements lie past 32 bits, adjusted in place."""
    torch = pytest.importorskip("torch")
    from chat_wgpu_b200 import GpuContext
    from chat_wgpu_b200.kernels import logits
    n, V = 29000, 151936  # 4.4e9 elements
    x = torch.zeros(n, V, dtype=torch.bfloat16, device="cuda")
    i = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    c = GpuContext(0, stream=torch.cuda.current_stream().cuda_stream)
    w = c.wrap(x)
    best = i([-1] * n)
    logits.AdjustLogits(c, logits=w, out=w, dtype="bf16", n_rows=n, vocab=V, best=c.wrap(best),
                        bias_tokens=c.wrap(i([(r * 7) % V for r in range(n)])),
                        bias_values=c.wrap(torch.full((n,), 2.0, device="cuda")),
                        bias_starts=c.wrap(i(list(range(n + 1)))), n_bias=n)()
    c.sync()
    want = (torch.arange(n, device="cuda") * 7) % V
    assert torch.equal(best.long(), want)
    for r in (0, 1, n // 2, n - 1):
        assert float(x[r, want[r]]) == 2.0 and float(x[r].float().sum()) == 2.0
    c.close()
    del x, w
    torch.cuda.empty_cache()


def test_far_slots():
    """Cache rows past 32-bit element offsets take the bits that near ones take."""
    torch = pytest.importorskip("torch")
    from chat_wgpu_b200 import GpuContext
    from chat_wgpu_b200.kernels import rope
    H, K, D, page, pages, T = 4, 8, 128, 64, 70000, 70
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(T, n * D, generator=g, device="cuda").bfloat16() for n in (H, K, K))
    kc, vc = (torch.empty(pages, K, page, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    i = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    c = GpuContext(0, stream=torch.cuda.current_stream().cuda_stream)
    one = torch.ones(D, device="cuda")
    for first in (0, pages - 2):
        rope.NormRope(c, plan=rope.rope_plan(c, D, 1e4), positions=c.wrap(i(list(range(T)))), dtype="bf16", n_tokens=T,
                      head_dim=D, eps=1e-6, n_heads=H, n_kv=K, q=c.wrap(q), q_norm=c.wrap(one),
                      q_out=c.wrap(torch.empty_like(q)), k=c.wrap(k), k_norm=c.wrap(one), v=c.wrap(v),
                      slots=c.wrap(i([first * page + t for t in range(T)])), k_cache=c.wrap(kc), v_cache=c.wrap(vc),
                      page_size=page, n_pages=pages)()
        c.sync()
    for x in (kc, vc):
        assert torch.equal(x[0], x[pages - 2]) and torch.equal(x[1, :, :6], x[pages - 1, :, :6])
        assert bool(x[0].isfinite().all())
    assert torch.equal(vc[0].transpose(0, 1).reshape(page, -1), v[:page])
    c.close()
    del kc, vc
    torch.cuda.empty_cache()
