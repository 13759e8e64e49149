"""Edges of the paged operators: shapes between the common ones, values that are not
finite, pages that are missing, captured steps, wrapped tensors."""
import subprocess
import sys

import numpy as np
import pytest

import paged_ref as ref
from conftest import ROOT
from test_gpu_paged import get, i32, tree_case, tree_run, tree_tolerance

pytestmark = pytest.mark.gpu


def attend(c, page, softcap=0.0, scale=None, gone=None, window=0):
    """The plain form over the keys a row sees, without those in gone[r] (bool per key)."""
    T, H, D = c["q"].shape
    K = c["kc"].shape[1]
    scale = D ** -0.5 if scale is None else scale
    out = np.zeros((T, H, D))
    big_s = big_v = 0.0
    for r in range(len(c["lens"])):
        a, b, n0 = int(c["starts"][r]), int(c["starts"][r + 1]), int(c["lens"][r])
        at = np.arange(n0 + b - a)
        pages = c["table"][r, at // page]
        where = np.concatenate([at[:n0], c["pos"][a:b]])
        for t in range(a, b):
            vis = np.concatenate([np.ones(n0, bool), c["see"][r][t - a]])
            if window:
                vis &= c["pos"][t] - where < window
            if gone is not None:
                vis &= ~gone[r]
            j = np.flatnonzero(vis)
            if not len(j):
                continue
            for h in range(H):
                k, v = (x[pages[j], h // (H // K), j % page] for x in (c["kc"], c["vc"]))
                with np.errstate(invalid="ignore"):
                    s = k @ c["q"][t, h] * scale
                fine = np.isfinite(s)
                if fine.any():
                    big_s = max(big_s, float((np.abs(k[fine]) @ np.abs(c["q"][t, h])).max()) * scale)
                big_v = max(big_v, float(np.abs(v[np.isfinite(v)]).max()))
                if softcap:
                    s = softcap * np.tanh(s / softcap)
                top = s.max()
                if top == -np.inf:
                    continue
                with np.errstate(invalid="ignore"):
                    w = np.exp(s - top)
                    out[t, h] = w @ v / w.sum()
    return out, big_s, big_v


# every kernel: f32; 16 bit with few rows; many rows; two row blocks; 256 dims in parts
KINDS = [  # dtype, heads, kv, dim, page, nodes
    ("f32", 4, 2, 64, 16, 5), ("f32", 16, 2, 128, 16, 9), ("bf16", 8, 2, 64, 16, 3), ("f16", 16, 4, 128, 16, 9),
    ("bf16", 16, 2, 128, 32, 12), ("f16", 16, 2, 64, 16, 30), ("bf16", 8, 4, 256, 8, 3), ("f16", 8, 4, 256, 16, 30),
]
kinds = pytest.mark.parametrize("kind", KINDS, ids=lambda k: "-".join(map(str, k)))


# ---------------------------------------------------------------- head dims
@pytest.mark.parametrize("case", [
    ("bf16", 16, 8, 16, [700, 130, 1], [8, 5, 1], {}), ("f16", 8, 4, 64, [3000], [40], {}),
    ("bf16", 8, 4, 8, [900, 40], [3, 9], {}), ("f16", 8, 4, 32, [1000], [30], dict(window=300, softcap=20.0)),
    ("bf16", 16, 8, 128, [5000], [1], {}), ("f16", 32, 8, 192, [500], [64], dict(empty=True)),
    ("bf16", 8, 4, 256, [777, 2], [100, 7], {})], ids=lambda c: f"{c[0]}-p{c[3]}-{max(c[4])}x{max(c[5])}")
def test_192_dims(ctx, case):
    dtype, H, K, page, lens, nodes, opt = case
    opt = dict(opt)
    c = tree_case(np.random.default_rng(sum(lens)), lens, nodes, dtype, H, K, 192, page, empty=opt.pop("empty", False))
    got = tree_run(ctx, c, dtype, H, K, 192, page, pad=8, off=8, **opt)
    want, s, v = attend(c, page, softcap=opt.get("softcap", 0.0), window=opt.get("window", 0))
    assert np.abs(got - want).max() <= tree_tolerance(dtype, s, v)
    ctx.sync()


@pytest.mark.parametrize("nodes", [3, 70])
def test_every_multiple_of_8(ctx, nodes):
    """All head dims that the tensor-core kernels take, of few rows and of many."""
    for D in range(8, 257, 8):
        dtype = "bf16" if D % 16 else "f16"
        c = tree_case(np.random.default_rng(D), [150, 20], [nodes, 2], dtype, 4, 2, D, 16)
        got = tree_run(ctx, c, dtype, 4, 2, D, 16)
        want, s, v = attend(c, 16)
        assert np.abs(got - want).max() <= tree_tolerance(dtype, s, v), D
        ctx.sync()


# ---------------------------------------------------------------- page plan
@pytest.mark.parametrize("n", [4079, 4080, 4096, 4097])
def test_plan_is_the_first_call(n):
    """Request counts around 48 KB of shared memory, each in a process of its own: no
    earlier call has raised the kernel's limit."""
    code = f"""
import sys
sys.path.insert(0, {ROOT!r})
import numpy as np
from chat_wgpu_b200 import GpuContext
from chat_wgpu_b200.kernels.pages import PagePlan
n = {n}
with GpuContext(0) as c:
    i = lambda a: c.storage_u32(np.ascontiguousarray(a, np.int32).view(np.uint32))
    out = dict(starts=i(np.zeros(n + 1)), positions=i(np.zeros(n)), slots=i(np.zeros(n)), owners=i(np.zeros(n)),
               used=i([0]))
    PagePlan(c, lens=i(np.full(n, 3)), news=i(np.ones(n)), free_pages=None, table=i(np.arange(n)), n_req=n,
             page_size=4, max_pages=1, n_free=0, max_tokens=n, **out)()
    assert np.array_equal(c.read_u32(out["slots"], n), np.arange(n) * 4 + 3)
    assert np.array_equal(c.read_u32(out["starts"], n + 1), np.arange(n + 1))
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("page", [4, 5])
def test_plan_marks_pages_that_lack(ctx, page):
    """Where the free list runs out, ids that an earlier step left in the table do not stay
    as if they were the request's: they become -1."""
    from chat_wgpu_b200.kernels.pages import PagePlan
    table = i32(ctx, [[7, 1, 2, 3], [4, 5, 6, 8], [9, 9, 9, 9]])
    out = {k: i32(ctx, np.full(s, -77)) for k, s in dict(starts=4, positions=20, slots=20, owners=20, used=1).items()}
    call = PagePlan(ctx, lens=i32(ctx, [3, 0, 1]), news=i32(ctx, [page, 2 * page + 1, 2]),
                    free_pages=i32(ctx, [11, 12]), table=table, n_req=3, page_size=page, max_pages=4, n_free=2,
                    max_tokens=20, **out)
    for _ in range(2):
        call()
        assert int(get(ctx, out["used"], 1)[0]) == 4
        assert get(ctx, table, 12).reshape(3, 4).tolist() == [[7, 11, 2, 3], [12, -1, -1, 8], [9, 9, 9, 9]]
        slots = get(ctx, out["slots"], 20)
        assert (slots[page:2 * page] == 12 * page + np.arange(page)).all()
        assert (slots[2 * page:3 * page + 1] == -1).all()
        assert (slots[3 * page + 1:3 * page + 3] == 9 * page + 1 + np.arange(2)).all()


@pytest.mark.parametrize("page", [4, 5])
def test_slots_past_31_bits(ctx, page):
    """A page id whose slots do not fit gets a slot that no cache has, so that the rows are
    reported where they are written, not stored elsewhere."""
    from chat_wgpu_b200.kernels.pages import PagePlan
    big = 2 ** 32 // page // 4 + 1  # times page: past 31 bits, and a small number in 32
    ids = [2 ** 30, 2 ** 31 - 1, big, 2 ** 31 // page]
    out = {k: i32(ctx, np.full(s, -77)) for k, s in dict(starts=5, positions=8, slots=8, owners=8, used=1).items()}
    PagePlan(ctx, lens=i32(ctx, [1, 1, 1, 1]), news=i32(ctx, [2, 2, 2, 2]), free_pages=None,
             table=i32(ctx, ids), n_req=4, page_size=page, max_pages=1, n_free=0, max_tokens=8, **out)()
    want = [min(p * page + 1 + j, 2 ** 31 - 1) for p in ids for j in range(2)]
    assert get(ctx, out["slots"], 8).tolist() == want


# ---------------------------------------------------------------- captured steps
def test_captured_step_outlives_larger_calls():
    """Plan, rotary and attention captured in a graph keep their results when the context
    later runs calls that need more scratch and another context takes scratch of its own
    and works beside the graph."""
    torch = pytest.importorskip("torch")
    from chat_wgpu_b200 import GpuContext
    from chat_wgpu_b200.kernels import pages, rope, tree
    side, beside = torch.cuda.Stream(), torch.cuda.Stream()
    g = torch.Generator(device="cuda").manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    i = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    H, K, page = 8, 2, 16

    def step(c, lens, n, D):
        """A request of `lens` tokens and n nodes: its calls and their result."""
        P = -(-(lens + n) // page)
        t = dict(lens=i([lens]), news=i([n]), free=i(list(range(P))), table=i([list(range(P))]),
                 starts=i([0, 0]), pos=i([0] * n), slots=i([0] * n), own=i([0] * n), used=i([0]), q=rnd(n, H * D),
                 k=rnd(n, K * D), v=rnd(n, K * D), kc=rnd(2 * P, K, page, D), vc=rnd(2 * P, K, page, D),
                 rot=torch.zeros(n, H * D, dtype=torch.bfloat16, device="cuda"),
                 out=torch.zeros(n, H * D, dtype=torch.bfloat16, device="cuda"))
        t["free"] += P
        w = {k: c.wrap(x) for k, x in t.items()}
        plan = rope.rope_plan(c, D, 1e4)
        return [pages.PagePlan(c, lens=w["lens"], news=w["news"], free_pages=w["free"], table=w["table"],
                               starts=w["starts"], positions=w["pos"], slots=w["slots"], owners=w["own"],
                               used=w["used"], n_req=1, page_size=page, max_pages=P, n_free=P, max_tokens=n),
                rope.RopeAppend(c, plan=plan, positions=w["pos"], dtype="bf16", n_tokens=n, n_heads=H, n_kv=K,
                                head_dim=D, q=w["q"], q_out=w["rot"], k=w["k"], v=w["v"], slots=w["slots"],
                                k_cache=w["kc"], v_cache=w["vc"], page_size=page, n_pages=2 * P),
                tree.TreeAttention(c, q=w["rot"], k_cache=w["kc"], v_cache=w["vc"], table=w["table"], lens=w["lens"],
                                   starts=w["starts"], out=w["out"], dtype="bf16", n_req=1, n_rows=n, max_nodes=n,
                                   n_heads=H, n_kv=K, head_dim=D, page_size=page, n_pages=2 * P, max_pages=P)], t["out"]

    c, other = GpuContext(0, stream=side.cuda_stream), GpuContext(0, stream=beside.cuda_stream)
    small, out = step(c, 5000, 3, 64)
    big, big_out = step(c, 9000, 60, 256)
    theirs, their_out = step(other, 9000, 3, 64)
    torch.cuda.synchronize()
    for f in small:
        f()
    side.synchronize()
    first = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        for f in small:
            f()
    for f in big + theirs:
        f()
    torch.cuda.synchronize()
    kept, many = (big_out.clone(), their_out.clone()), []
    for _ in range(40):
        with torch.cuda.stream(side):
            out.zero_()
            graph.replay()
            many.append((out.clone(), first))
        with torch.cuda.stream(beside):
            theirs[2]()
            many.append((their_out.clone(), kept[1]))
    for f in big:
        f()
    torch.cuda.synchronize()
    assert torch.equal(big_out, kept[0]) and bool((first != 0).any())
    assert all(torch.equal(a, b) for a, b in many)
    c.sync()
    other.sync()
    del graph
    c.close()
    other.close()


# ---------------------------------------------------------------- values that are not finite
@kinds
@pytest.mark.parametrize("lens", [[40, 3], [9000, 3]], ids=["whole", "cut"])
def test_query_of_nan(ctx, kind, lens):
    """A row whose scores are NaN is NaN, whether its item is cut or not; the others stay."""
    dtype, H, K, D, page, n = kind
    c = tree_case(np.random.default_rng(21), lens, [n, 2], dtype, H, K, D, page, poison=False)
    want, s, v = attend(c, page)
    c["q"][1, H - 1, 5] = np.nan
    got = tree_run(ctx, c, dtype, H, K, D, page)
    assert np.isnan(got[1, H - 1]).all()
    rest = np.ones(got.shape[:2], bool)
    rest[1, H - 1] = False
    assert np.abs(got - want)[rest].max() <= tree_tolerance(dtype, s, v)
    ctx.sync()


@pytest.mark.parametrize("kind", [k for k in KINDS if k[0] != "f32"], ids=lambda k: "-".join(map(str, k)))
@pytest.mark.parametrize("lens", [[400, 3], [9000, 3]], ids=["whole", "cut"])
def test_scores_of_minus_infinity(ctx, kind, lens):
    """Keys that score -inf weigh nothing, first tiles full of them included; a row with
    no other key gives zeros."""
    dtype, H, K, D, page, n = kind
    c = tree_case(np.random.default_rng(22), lens, [n, 2], dtype, H, K, D, page, poison=False)
    c["q"][:, :, 2] = 1.0
    at = np.arange(320)
    c["kc"][c["table"][0, at // page], :, at % page, 2] = -np.inf
    every = np.arange(5)  # all keys of the second request
    c["kc"][c["table"][1, every // page], :, every % page, 2] = -np.inf
    got = tree_run(ctx, c, dtype, H, K, D, page)
    want, s, v = attend(c, page)
    assert (got[n:] == 0).all()
    assert np.abs(got - want).max() <= tree_tolerance(dtype, s, v)
    ctx.sync()


@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (16, 2, 128), (8, 4, 256)])
def test_many_tiles_of_values_that_are_not_finite(ctx, heads, kv, dim):
    """f32, one tile after another holding values that no row sees and that are not finite: every
    tile's rows use that tile's own sets."""
    c = tree_case(np.random.default_rng(24), [30, 0], [400, 3], "f32", heads, kv, dim, 16, poison=False)
    m = 400
    for j in range(0, m, 3):  # node j: seen by nobody
        c["see"][0][:, j] = False
        c["vc"][c["table"][0, (30 + j) // 16], :, (30 + j) % 16] = np.nan if j % 2 else np.inf
    words = c["mask"].shape[1]
    bits = np.zeros((c["T"], words * 32), np.uint8)
    bits[:m, :m] = c["see"][0]
    bits[m:, :3] = c["see"][1]
    c["mask"] = np.packbits(bits, axis=1, bitorder="little").view(np.uint32)
    want, s, v = attend(c, 16)
    for _ in range(5):
        got = tree_run(ctx, c, "f32", heads, kv, dim, 16)
        assert np.abs(got - want).max() <= tree_tolerance("f32", s, v)
    ctx.sync()


@pytest.mark.parametrize("kind", [k for k in KINDS if k[0] == "f32"], ids=lambda k: "-".join(map(str, k)))
@pytest.mark.parametrize("lens", [[400, 3], [9000, 3]], ids=["whole", "cut"])
def test_f32_scores_of_minus_infinity(ctx, kind, lens):
    test_scores_of_minus_infinity(ctx, kind, lens)


@kinds
def test_values_of_infinity_in_the_prefix(ctx, kind):
    """An infinite value that every row sees comes out infinite in its dim, and a score of
    +inf makes its row NaN; other dims and rows stay."""
    dtype, H, K, D, page, n = kind
    c = tree_case(np.random.default_rng(23), [700], [n], dtype, H, K, D, page, poison=False)
    c["vc"][c["table"][0, 100 // page], :, 100 % page, 4] = np.inf
    c["vc"][c["table"][0, 130 // page], :, 130 % page, 7] = -np.inf
    got = tree_run(ctx, c, dtype, H, K, D, page, scale=0.01)
    want, s, v = attend(c, page, scale=0.01)
    assert (got[:, :, 4] == np.inf).all() and (got[:, :, 7] == -np.inf).all()
    rest = np.ones(D, bool)
    rest[[4, 7]] = False
    assert np.abs(got[:, :, rest] - want[:, :, rest]).max() <= tree_tolerance(dtype, s, v)
    c["kc"][c["table"][0, 300 // page], :, 300 % page, 2] = np.inf
    c["q"][:, :, 2] = -1.0
    c["q"][0, :, 2] = 1.0    # +inf for row 0, -inf for the others
    got = tree_run(ctx, c, dtype, H, K, D, page, scale=0.01)
    want, s, v = attend(c, page, scale=0.01)
    assert np.isnan(got[0]).all()
    assert (got[1:, :, 4] == np.inf).all() and (got[1:, :, 7] == -np.inf).all()
    assert np.abs(got[1:, :, rest] - want[1:, :, rest]).max() <= tree_tolerance(dtype, s, v)
    ctx.sync()


# ---------------------------------------------------------------- pages that are missing
def tree_reported(ctx, c, dtype, *shape, **opt):
    """tree_run of a call that reports its input: the rows, and the report."""
    from chat_wgpu_b200 import CwError
    seen, read = [], ref.read

    def after(ctx_, buf, dtype_, size):
        with pytest.raises(CwError) as e:
            ctx_.sync()
        seen.append(e.value.status)
        return read(ctx_, buf, dtype_, size)

    ref.read = after
    try:
        return tree_run(ctx, c, dtype, *shape, **opt), seen[0]
    finally:
        ref.read = read


@kinds
@pytest.mark.parametrize("ctx_len", [330, 9000])
def test_unusable_pages(ctx, kind, ctx_len):
    """Keys of a page id outside the cache weigh nothing and are reported; other requests'
    rows are as ever."""
    dtype, H, K, D, page, n = kind
    c = tree_case(np.random.default_rng(31), [ctx_len, 50, 300], [n, 2, n], dtype, H, K, D, page, poison=False)
    good, s0, v0 = attend(c, page)
    gone = [np.zeros(ctx_len + n, bool), np.zeros(52, bool), np.zeros(300 + n, bool)]
    lost = [(0, 3, -1), (0, 4, c["n_pages"]), (2, 0, 2 ** 31 - 1), (2, 300 // page, -7)]
    sent = dict(c, table=c["table"].copy())
    for r, p, bad in lost:
        sent["table"][r, p] = bad
        gone[r][p * page:(p + 1) * page] = True
    got, status = tree_reported(ctx, sent, dtype, H, K, D, page)
    assert status == 1
    ctx.sync()
    want, s, v = attend(c, page, gone=gone)
    tol = tree_tolerance(dtype, max(s, s0), max(v, v0))
    assert np.abs(got - want).max() <= tol
    assert np.abs(got - good)[n:n + 2].max() <= tol


@pytest.mark.parametrize("case", [("f32", 8, 2, 64, 8, 70), ("bf16", 8, 2, 64, 8, 70), ("f16", 8, 1, 128, 128, 40),
                                  ("bf16", 8, 4, 256, 32, 100), ("bf16", 4, 2, 72, 16, 9)],
                         ids=lambda c: "-".join(map(str, c)))
def test_one_page_in_three(ctx, case):
    """Many missing pages over many tiles, some tiles without any page; no key at all."""
    dtype, H, K, D, page, n = case
    rng = np.random.default_rng(33)
    c = tree_case(rng, [3000, 1500, 70], [n, 1, 2], dtype, H, K, D, page)
    gone, sent = [], dict(c, table=c["table"].copy())
    for r in range(3):
        lost = rng.random(c["max_pages"]) < (1.0 if r == 2 else 0.33)
        lost[512 // page:1024 // page] |= r == 0
        sent["table"][r, lost] = -1
        gone.append(np.repeat(lost, page)[:c["lens"][r] + c["starts"][r + 1] - c["starts"][r]])
    got, status = tree_reported(ctx, sent, dtype, H, K, D, page, softcap=9.0)
    assert status == 1
    want, s, v = attend(c, page, gone=gone, softcap=9.0)
    assert (got[-2:] == 0).all()
    assert np.abs(got - want).max() <= tree_tolerance(dtype, s, v)


@kinds
def test_pages_given_up_before_the_window(ctx, kind):
    """Pages whose keys no row can see need not be there, nor are they reported, where the
    window's edge lies inside a tile."""
    dtype, H, K, D, page, n = kind
    window = 64 + page + 3
    lens = 1024 + 2 * page + 5 + window  # the first key that a row sees: 1024 + 2 * page + 6
    c = tree_case(np.random.default_rng(32), [lens], [n], dtype, H, K, D, page, poison=False)
    want, s, v = attend(c, page, window=window)
    sent = dict(c, table=c["table"].copy())
    sent["table"][0, :(lens - window + 1) // page] = -1
    got = tree_run(ctx, sent, dtype, H, K, D, page, window=window)
    ctx.sync()
    assert np.abs(got - want).max() <= tree_tolerance(dtype, s, v)


# ---------------------------------------------------------------- weights in 16 bits
@pytest.mark.parametrize("kind", [k for k in KINDS if k[0] == "f16"], ids=lambda k: "-".join(map(str, k)))
def test_a_dominating_key(ctx, kind):
    """A first key e^17.5 above the other 30000, whose joint share is 7.5e-4: the value is 0
    at that key and 1 elsewhere, so the share is the result.  All requests' tables name the
    same three pages; there are enough requests that items are whole."""
    dtype, H, K, D, page, n = kind
    lens, req = 30000, 160
    pages = -(-(lens + n) // page)
    kc, vc = np.zeros((3, K, page, D)), np.ones((3, K, page, D))
    kc[1, :, 0, 0], vc[1, :, 0] = 17.5, 0.0
    table = np.zeros((req, pages), np.int32)
    table[:, 0] = 1
    q = np.zeros((req * n, H, D))
    q[:, :, 0] = 1.0
    c = dict(lens=np.full(req, lens), starts=np.arange(req + 1) * n, T=req * n, N=n, table=table, kc=kc, vc=vc,
             pos=np.zeros(req * n, np.int32), q=q, max_pages=pages, n_pages=3)
    got = tree_run(ctx, c, dtype, H, K, D, page, scale=1.0, mask=False)
    share = (lens + np.arange(n)) * np.exp(-17.5)  # node i sees nodes 0..i; one of the prefix is the large one
    want = np.tile(share / (1 + share), req)[:, None, None]
    # the largest weight is 2^7 at least, so f16's fixed step of 2^-24 below 2^-14 moves a
    # weight by at most 2^-25 / 2^7 of it; the sum takes the same rounded weights.  Then
    # f32 arithmetic and one rounding of the result.
    assert np.abs(got - want).max() <= (lens + n) * 2.0 ** -32 + (ref.UNIT["f16"] + 1e-5) * want.max()
    ctx.sync()


@kinds
@pytest.mark.parametrize("lens", [[400, 3], [9000, 3]], ids=["whole", "cut"])
def test_no_weight_times_infinity(ctx, kind, lens):
    """A key that scores -inf weighs 0, and 0 times an infinite value is NaN, wherever the
    key's tile was dealt to; other dims stay."""
    dtype, H, K, D, page, n = kind
    c = tree_case(np.random.default_rng(25), lens, [n, 2], dtype, H, K, D, page, poison=False)
    c["q"][:, :, 2] = 1.0
    at = np.arange(320)
    c["kc"][c["table"][0, at // page], :, at % page, 2] = -np.inf
    c["vc"][c["table"][0, 100 // page], :, 100 % page, 4] = np.inf
    got = tree_run(ctx, c, dtype, H, K, D, page)
    want, s, v = attend(c, page)
    assert np.isnan(want[:n, :, 4]).all() and np.isnan(got[:n, :, 4]).all()
    fine = np.isfinite(want)
    assert np.abs(got[fine] - want[fine]).max() <= tree_tolerance(dtype, s, v)
    ctx.sync()
