"""Greedy decode with drafted token trees over a paged cache.

One step runs every session's open tokens and a small tree of drafted ones
together: cw_page_plan gives the rows their pages, and per layer cw_rope_append
writes their keys and values and cw_tree_attention lets each node see its
session's cached tokens and its own ancestors.  The drafted nodes that the model
would have produced itself are kept, so the tokens are those of plain greedy decode
(model.generate_op_by_op) in fewer steps.  Drafts come from the session's own text:
what followed the last occurrences of its last tokens.

    python -m chat_wgpu_b200.treedecode model.gguf 1 5 9 2 --new 32
"""
from __future__ import annotations

import numpy as np

from .kernels import activation, argmax, attention, norm, pages, q4, rope, tree
from .model import OpByOpQwen3


def lookup_draft(tokens, width: int = 2, depth: int = 4, match: int = 2) -> list[tuple[int, int]]:
    """Nodes (parent, token) drafted after `tokens`, parents before children, parent
    -1 = the last token: the continuations of up to `width` earlier places where the
    last `match` tokens occur, up to `depth` tokens each, shared prefixes merged."""
    nodes: list[tuple[int, int]] = []
    child: dict[tuple[int, int], int] = {}
    tail = list(tokens[-match:])
    starts = [i for i in range(len(tokens) - match - 1, -1, -1) if list(tokens[i:i + match]) == tail]
    for i in starts[:width]:
        at = -1
        for t in tokens[i + match:i + match + depth]:
            if (at, t) not in child:
                child[at, t] = len(nodes)
                nodes.append((at, int(t)))
            at = child[at, t]
    return nodes


class Session:
    """One request: its tokens, how many of them are stored in order in the cache,
    and the last token that no step has run yet."""

    def __init__(self, prompt):
        self.tokens = [int(t) for t in prompt]
        self.stored = 0
        self.n_prompt = len(self.tokens)

    @property
    def produced(self) -> list[int]:
        return self.tokens[self.n_prompt:]


class TreeDecoder:
    """Several sessions of one OpByOpQwen3 stepped together."""

    def __init__(self, model: OpByOpQwen3, prompts, max_seq: int, page_size: int = 16,
                 chunk: int = 64, draft=lookup_draft):
        if not prompts or any(len(p) == 0 for p in prompts):
            raise ValueError("every session needs a prompt")
        if not 1 <= chunk <= 1024:
            raise ValueError(f"chunk {chunk}: rows of a session in a step, 1..1024")
        self.m, self.ctx, self.page, self.chunk, self.draft = model, model.ctx, page_size, chunk, draft
        self.sessions = [Session(p) for p in prompts]
        self.max_seq = max_seq
        n = len(self.sessions)
        # room for the drafts of one step past max_seq
        self.max_pages = -(-(max_seq + chunk) // page_size)
        self.n_pages = n * self.max_pages
        kvd = model.n_kv_heads * model.head_dim
        self.cache = [(self.ctx.empty_persistent(self.n_pages * page_size * kvd),
                       self.ctx.empty_persistent(self.n_pages * page_size * kvd))
                      for _ in range(model.n_layers)]
        self.table = self._i32(np.full((n, self.max_pages), -1))
        self.plan = rope.rope_plan(self.ctx, model.head_dim, model.rope_theta)
        self.steps = 0

    def close(self) -> None:
        for k, v in self.cache:
            k.release()
            v.release()
        for b in (self.table, self.plan):
            b.release()
        self.cache = []

    def _i32(self, a):
        return self.ctx.storage_u32(np.ascontiguousarray(a, np.int32).view(np.uint32))

    def _free_pages(self) -> np.ndarray:
        """Pages that hold no token stored in order (the last step's drafts are given up)."""
        rows = self.ctx.read_u32(self.table, len(self.sessions) * self.max_pages).view(np.int32)
        rows = rows.reshape(len(self.sessions), -1)
        held = [rows[i, :-(-s.stored // self.page)] for i, s in enumerate(self.sessions)]
        return np.setdiff1d(np.arange(self.n_pages), np.concatenate(held))

    def _forward(self, rows, lens, news, depths, see):
        """Logits [rows, vocab] buffer of the step's nodes."""
        m, ctx, T, n = self.m, self.ctx, len(rows), len(lens)
        free = self._free_pages()
        most = int(news.max())
        words = -(-most // 32)
        bits = np.zeros((T, words * 32), np.uint8)
        start = 0
        for r in range(n):
            bits[start:start + news[r], :news[r]] = see[r]
            start += int(news[r])
        temp = [self._i32(a) for a in (lens, news, free, depths)]
        outs = [self._i32(np.zeros(k)) for k in (n + 1, T, T, T, 1)]
        mask = ctx.storage_u32(np.packbits(bits, axis=1, bitorder="little").view(np.uint32))
        starts, pos, slots, owners, used = outs
        pages.PagePlan(ctx, lens=temp[0], news=temp[1], free_pages=temp[2], table=self.table,
                       depths=temp[3], starts=starts, positions=pos, slots=slots, owners=owners,
                       used=used, n_req=n, page_size=self.page, max_pages=self.max_pages,
                       n_free=len(free), max_tokens=T)()
        nh, nkv, hd, dim = m.n_heads, m.n_kv_heads, m.head_dim, m.dim
        x = ctx.empty(T * dim)
        for i, t in enumerate(rows):
            ctx.copy(m.embed_tbl, int(t) * dim, x, i * dim, dim)

        def proj(w, a):
            buf, in_f, out_f = w
            return q4.q4_0_gemm(ctx, a, buf, T, in_f, out_f)

        for l, (kc, vc) in zip(m.layers, self.cache):
            a = norm.rmsnorm(ctx, x, l["attn_norm"], T, dim, m.eps)
            q = norm.rmsnorm(ctx, proj(l["wq"], a), l["q_norm"], T * nh, hd, m.eps)
            k = norm.rmsnorm(ctx, proj(l["wk"], a), l["k_norm"], T * nkv, hd, m.eps)
            rope.RopeAppend(ctx, plan=self.plan, positions=pos, dtype="f32", n_tokens=T,
                            n_heads=nh, n_kv=nkv, head_dim=hd, q=q, q_out=q, k=k,
                            v=proj(l["wv"], a), slots=slots, k_cache=kc, v_cache=vc,
                            page_size=self.page, n_pages=self.n_pages)()
            o = ctx.empty(T * nh * hd)
            tree.TreeAttention(ctx, q=q, k_cache=kc, v_cache=vc, table=self.table, lens=temp[0],
                               starts=starts, mask=mask, out=o, dtype="f32", n_req=n, n_rows=T,
                               max_nodes=most, n_heads=nh, n_kv=nkv, head_dim=hd,
                               page_size=self.page, n_pages=self.n_pages,
                               max_pages=self.max_pages)()
            x = attention.add(ctx, x, proj(l["wo"], o), T * dim)
            a = norm.rmsnorm(ctx, x, l["ffn_norm"], T, dim, m.eps)
            act = activation.swiglu(ctx, proj(l["gate"], a), proj(l["up"], a), T * m.hidden)
            x = attention.add(ctx, x, proj(l["down"], act), T * dim)
        logits = proj(m.lm_head, norm.rmsnorm(ctx, x, m.final_norm, T, dim, m.eps))
        for b in temp + outs + [mask]:
            b.release()
        return logits

    def step(self, max_new: int, want_logits: bool = False):
        """One step of every session that still has tokens to produce; with
        want_logits the logits that each newly produced token was chosen from."""
        ctx, vocab = self.ctx, self.m.vocab
        rows, lens, news, depths, see, trees = [], [], [], [], [], []
        for s in self.sessions:
            open_ = s.tokens[s.stored:s.stored + self.chunk]
            done = len(s.produced) >= max_new
            drafts = []
            if done:
                open_ = []
            elif s.stored + len(open_) == len(s.tokens):
                room = min(self.chunk - len(open_), self.max_seq - len(s.tokens))
                drafts = self.draft(s.tokens)[:max(room, 0)]
            c, m = len(open_), len(open_) + len(drafts)
            v = np.zeros((m, m), bool)
            depth = list(range(c))
            for i in range(c):
                v[i, :i + 1] = True
            for j, (parent, _) in enumerate(drafts):
                up = c - 1 if parent < 0 else c + parent
                v[c + j] = v[up]
                v[c + j, c + j] = True
                depth.append(depth[up] + 1)
            rows += open_ + [t for _, t in drafts]
            lens.append(s.stored)
            news.append(m)
            depths += depth
            see.append(v)
            trees.append((c, drafts))
        if not rows:
            return []
        ctx.reset_frame()
        lens, news = np.array(lens), np.array(news)
        logits = self._forward(rows, lens, news, np.array(depths), see)
        self.steps += 1
        best = np.empty(len(rows), np.int64)
        row = ctx.empty(vocab)
        for i in range(len(rows)):
            ctx.copy(logits, i * vocab, row, 0, vocab)
            best[i] = ctx.read_u32(argmax.argmax(ctx, row, vocab), 1)[0]
        out, first = [], 0
        for s, (c, drafts), m in zip(self.sessions, trees, news):
            base, first = first, first + int(m)
            if not m:
                continue
            s.stored += c
            if s.stored < len(s.tokens):  # a prompt in pieces: nothing is produced yet
                continue
            at, kept = c - 1, 0
            while len(s.produced) < max_new:
                token = int(best[base + at])
                if want_logits:
                    ctx.copy(logits, (base + at) * vocab, row, 0, vocab)
                    out.append((s, len(s.produced), ctx.read(row, vocab)))
                s.tokens.append(token)
                nxt = [j for j, (p, t) in enumerate(drafts)
                       if t == token and (c - 1 if p < 0 else c + p) == at]
                if not nxt:
                    break
                at = c + nxt[0]
                if at == c + kept:  # right after the kept ones: stored in order
                    kept += 1
            s.stored += kept
        return out

    def generate(self, max_new: int) -> list[list[int]]:
        """max_new greedy tokens of every session."""
        if any(s.n_prompt + max_new > self.max_seq for s in self.sessions):
            raise ValueError("prompt + max_new exceeds max_seq")
        while any(len(s.produced) < max_new for s in self.sessions):
            self.step(max_new)
        return [s.produced for s in self.sessions]


def main() -> None:
    import argparse

    from .context import GpuContext
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("model")
    ap.add_argument("prompt", nargs="+", type=int)
    ap.add_argument("--new", type=int, default=32)
    a = ap.parse_args()
    with GpuContext(0) as ctx:
        d = TreeDecoder(OpByOpQwen3(ctx, a.model), [a.prompt], len(a.prompt) + a.new)
        print(*d.generate(a.new)[0])
        print(f"{a.new} tokens in {d.steps} steps")
        d.close()


if __name__ == "__main__":
    main()
