"""Greedy decode with drafted token trees over a paged cache.

One step runs every session's open tokens and a small tree of drafted ones
together: cw_page_plan gives the rows their pages, and per layer cw_rope_append
writes their keys and values and cw_tree_attention lets each node see its
session's cached tokens and its own ancestors.  The drafted nodes that the model
would have produced itself are kept, so the tokens are those of plain greedy decode
(model.generate_op_by_op) in fewer steps.  Drafts come from the session's own text:
what followed the last occurrences of its last tokens.

TreeDecoder.prefill takes whole prompts in at once, each of its own length up to max_seq: per
layer cw_norm_rope writes their keys and values and cw_prompt_attention lets each token see
its own prompt up to itself.  With penalties, biases or a set of allowed tokens
cw_adjust_logits chooses the step's tokens.

    python -m chat_wgpu_b200.treedecode model.gguf 1 5 9 2 --new 32 --prefill --repetition 1.1
"""
from __future__ import annotations

import numpy as np

from .kernels import (activation, argmax, attention, logits as rules, norm, pages, prompt, q4, rope,
                      tree)
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
    """Several sessions of one OpByOpQwen3 stepped together.  penalties = (repetition,
    frequency, presence), biases = {token: value} and allowed = token ids (None: all) apply
    to every session's logits; the repetition penalty counts the prompt, too."""

    def __init__(self, model: OpByOpQwen3, prompts, max_seq: int, page_size: int = 16,
                 chunk: int = 64, draft=lookup_draft, penalties=None, biases=None, allowed=None):
        if not prompts or any(len(p) == 0 for p in prompts):
            raise ValueError("every session needs a prompt")
        if not 1 <= chunk <= 1024:
            raise ValueError(f"chunk {chunk}: rows of a session in a step, 1..1024")
        if allowed is not None:
            allowed = np.array(sorted(allowed), np.int64)
            if allowed.size == 0 or allowed[0] < 0 or allowed[-1] >= model.vocab:
                raise ValueError(f"allowed: at least one token, each in 0..{model.vocab - 1}")
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
        self.penalties, self.biases, self.mask = penalties, dict(biases or {}), None
        if allowed is not None:
            bits = np.zeros(-(-model.vocab // 32) * 32, np.uint8)
            bits[allowed] = 1
            self.mask = self.ctx.storage_u32(np.packbits(bits, bitorder="little").view(np.uint32))

    def close(self) -> None:
        for k, v in self.cache:
            k.release()
            v.release()
        for b in (self.table, self.plan, self.mask):
            if b is not None:
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

    def _place(self, lens, news, T, depths=None):
        """Pages, positions and slots of a step's T rows; the buffers, to be released."""
        ctx, n = self.ctx, len(lens)
        free = self._free_pages()
        given = [self._i32(a) for a in (lens, news, free)]
        deep = None if depths is None else self._i32(depths)
        out = {k: self._i32(np.zeros(c)) for k, c in dict(starts=n + 1, positions=T, slots=T,
                                                          owners=T, used=1).items()}
        pages.PagePlan(ctx, lens=given[0], news=given[1], free_pages=given[2], table=self.table,
                       depths=deep, n_req=n, page_size=self.page, max_pages=self.max_pages,
                       n_free=len(free), max_tokens=T, **out)()
        out.update(lens=given[0], news=given[1], free=given[2])
        if deep is not None:
            out["depths"] = deep
        return out

    def _layers(self, rows, attend, x=None):
        """Hidden rows of the tokens after the layers; attend(q, k, v, layer, cache) gives the
        attention's rows.  With x, a buffer of their own for the rows, each layer is a frame:
        the activations of one are held at a time, not of all."""
        m, ctx, T = self.m, self.ctx, len(rows)
        dim = m.dim
        own = x
        if own is None:
            x = ctx.empty(T * dim)
        for i, t in enumerate(rows):
            ctx.copy(m.embed_tbl, int(t) * dim, x, i * dim, dim)
        for l, cache in zip(m.layers, self.cache):
            a = norm.rmsnorm(ctx, x, l["attn_norm"], T, dim, m.eps)
            o = attend(self._proj(l["wq"], a, T), self._proj(l["wk"], a, T),
                       self._proj(l["wv"], a, T), l, cache)
            x = attention.add(ctx, x, self._proj(l["wo"], o, T), T * dim)
            a = norm.rmsnorm(ctx, x, l["ffn_norm"], T, dim, m.eps)
            act = activation.swiglu(ctx, self._proj(l["gate"], a, T), self._proj(l["up"], a, T),
                                    T * m.hidden)
            x = attention.add(ctx, x, self._proj(l["down"], act, T), T * dim)
            if own is not None:
                ctx.copy(x, 0, own, 0, T * dim)
                ctx.reset_frame()
                x = own
        return x

    def _proj(self, w, a, T):
        buf, in_f, out_f = w
        return q4.q4_0_gemm(self.ctx, a, buf, T, in_f, out_f)

    def _forward(self, rows, lens, news, depths, see):
        """Logits [rows, vocab] buffer of the step's nodes."""
        m, ctx, T, n = self.m, self.ctx, len(rows), len(lens)
        nh, nkv, hd = m.n_heads, m.n_kv_heads, m.head_dim
        most = int(news.max())
        words = -(-most // 32)
        bits = np.zeros((T, words * 32), np.uint8)
        start = 0
        for r in range(n):
            bits[start:start + news[r], :news[r]] = see[r]
            start += int(news[r])
        at = self._place(lens, news, T, depths)
        mask = ctx.storage_u32(np.packbits(bits, axis=1, bitorder="little").view(np.uint32))

        def attend(q, k, v, l, cache):
            kc, vc = cache
            q = norm.rmsnorm(ctx, q, l["q_norm"], T * nh, hd, m.eps)
            k = norm.rmsnorm(ctx, k, l["k_norm"], T * nkv, hd, m.eps)
            rope.RopeAppend(ctx, plan=self.plan, positions=at["positions"], dtype="f32", n_tokens=T,
                            n_heads=nh, n_kv=nkv, head_dim=hd, q=q, q_out=q, k=k, v=v,
                            slots=at["slots"], k_cache=kc, v_cache=vc, page_size=self.page,
                            n_pages=self.n_pages)()
            o = ctx.empty(T * nh * hd)
            tree.TreeAttention(ctx, q=q, k_cache=kc, v_cache=vc, table=self.table, lens=at["lens"],
                               starts=at["starts"], mask=mask, out=o, dtype="f32", n_req=n, n_rows=T,
                               max_nodes=most, n_heads=nh, n_kv=nkv, head_dim=hd,
                               page_size=self.page, n_pages=self.n_pages,
                               max_pages=self.max_pages)()
            return o

        x = self._layers(rows, attend)
        logits = self._proj(m.lm_head, norm.rmsnorm(ctx, x, m.final_norm, T, m.dim, m.eps), T)
        for b in list(at.values()) + [mask]:
            b.release()
        return logits

    def prefill(self) -> None:
        """The prompts of the sessions that no step has run yet, but for their last tokens, in
        one pass: packed rows, each prompt's own length.  It holds one layer's activations of
        all rows, 4 bytes times 7 dim + 3 hidden + 2 n_heads * head_dim + 3 n_kv_heads * head_dim
        a token, and the attention's scratch (cw_prompt_attention)."""
        m, ctx = self.m, self.ctx
        nh, nkv, hd = m.n_heads, m.n_kv_heads, m.head_dim
        if any(s.n_prompt > self.max_seq for s in self.sessions):
            raise ValueError("a prompt exceeds max_seq")
        news = np.array([0 if s.stored else s.n_prompt - 1 for s in self.sessions])
        T, n = int(news.sum()), len(news)
        if T == 0:
            return
        ctx.reset_frame()
        at = self._place(np.array([s.stored for s in self.sessions]), news, T)

        def attend(q, k, v, l, cache):
            k_rows, o = ctx.empty(T * nkv * hd), ctx.empty(T * nh * hd)
            rope.NormRope(ctx, plan=self.plan, positions=at["positions"], dtype="f32", n_tokens=T,
                          head_dim=hd, eps=m.eps, n_heads=nh, n_kv=nkv, q=q, q_norm=l["q_norm"],
                          q_out=q, k=k, k_norm=l["k_norm"], k_out=k_rows, v=v, slots=at["slots"],
                          k_cache=cache[0], v_cache=cache[1], page_size=self.page,
                          n_pages=self.n_pages)()
            prompt.PromptAttention(ctx, q=q, k=k_rows, v=v, starts=at["starts"], out=o, dtype="f32",
                                   n_req=n, n_rows=T, n_heads=nh, n_kv=nkv, head_dim=hd)()
            return o

        try:
            at["x"] = ctx.empty_persistent(T * m.dim)
            self._layers([t for s, c in zip(self.sessions, news) for t in s.tokens[:c]], attend,
                         at["x"])
            ctx.sync()
        finally:
            for b in at.values():
                b.release()
        for s, c in zip(self.sessions, news):
            s.stored += int(c)

    def _choose(self, logits, histories, leads):
        """The token of each row of logits, which become the adjusted ones; without penalties
        the histories are not read."""
        ctx, T, vocab = self.ctx, len(histories), self.m.vocab
        flat = lambda lists: [x for y in lists for x in y]  # noqa: E731
        begin = lambda lists: np.concatenate([[0], np.cumsum([len(x) for x in lists])])  # noqa: E731
        temp, more = {}, {}
        if self.penalties is not None:
            temp.update(penalties=ctx.storage(np.tile(np.float32(self.penalties), (T, 1))),
                        tokens=self._i32(flat(histories)), starts=self._i32(begin(histories)),
                        prompts=self._i32(leads))
            more["n_tokens"] = sum(map(len, histories))
        if self.biases:
            pairs = [list(self.biases)] * T
            temp.update(bias_tokens=self._i32(flat(pairs)), bias_starts=self._i32(begin(pairs)),
                        bias_values=ctx.storage(np.tile(np.float32(list(self.biases.values())), T)))
            more["n_bias"] = len(self.biases) * T
        if self.mask is not None:
            temp["mask_rows"] = self._i32(np.zeros(T))
            more.update(masks=self.mask, n_masks=1)
        temp["best"] = self._i32(np.zeros(T))
        rules.AdjustLogits(ctx, logits=logits, out=logits, dtype="f32", n_rows=T, vocab=vocab, **temp,
                           **more)()
        best = ctx.read_u32(temp["best"], T).astype(np.int64)
        for b in temp.values():
            b.release()
        return best

    def step(self, max_new: int, want_logits: bool = False):
        """One step of every session that still has tokens to produce; with
        want_logits the logits that each newly produced token was chosen from."""
        ctx, vocab = self.ctx, self.m.vocab
        rows, lens, news, depths, see, trees = [], [], [], [], [], []
        histories, leads = [], []
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
            # histories of the rows that tokens are picked from, the last open one and the drafts
            counted = self.penalties is not None and c > 0 and s.stored + c == len(s.tokens)
            text = [[] for _ in range(m)]
            if counted:
                text[c - 1] = list(s.tokens)
            for i in range(c):
                v[i, :i + 1] = True
            for j, (parent, token) in enumerate(drafts):
                up = c - 1 if parent < 0 else c + parent
                v[c + j] = v[up]
                v[c + j, c + j] = True
                depth.append(depth[up] + 1)
                if counted:
                    text[c + j] = text[up] + [token]
            histories += text
            leads += [s.n_prompt] * m
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
        row = ctx.empty(vocab)
        if self.penalties is not None or self.biases or self.mask is not None:
            best = self._choose(logits, histories, leads)
        else:
            best = np.empty(len(rows), np.int64)
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
    ap.add_argument("--prefill", action="store_true", help="take the prompt in as one pass")
    ap.add_argument("--repetition", type=float, default=1.0)
    ap.add_argument("--frequency", type=float, default=0.0)
    ap.add_argument("--presence", type=float, default=0.0)
    a = ap.parse_args()
    penalties = (a.repetition, a.frequency, a.presence)
    with GpuContext(0) as ctx:
        d = TreeDecoder(OpByOpQwen3(ctx, a.model), [a.prompt], len(a.prompt) + a.new,
                        penalties=None if penalties == (1.0, 0.0, 0.0) else penalties)
        if a.prefill:
            d.prefill()
        print(*d.generate(a.new)[0])
        print(f"{a.new} tokens in {d.steps} steps")
        d.close()


if __name__ == "__main__":
    main()
