"""Stand-ins for the kernels of drafted tokens, with torch on the CPU, beside those of emulated_kernels.py and
emulated_beams.py."""
from __future__ import annotations

import torch

import emulated_beams


def attention_tree(q, out, num_heads, num_kv_heads, head_dim, k_cache, v_cache, page_size, block_tables, context_lens, q_start,
                   seen, scale, window, max_nodes, max_context):
    group = num_heads // num_kv_heads
    scale = float(torch.tensor(scale, dtype=torch.float32))
    for b in range(block_tables.shape[0]):
        t0, t1 = int(q_start[b]), int(q_start[b + 1])
        n, base = t1 - t0, int(context_lens[b]) - (t1 - t0)
        assert n <= max_nodes and base + n <= max_context
        for t in range(t0, t1):
            bits = int(seen[t]) & (1 << n) - 1
            first = max(0, base + bin(bits).count("1") - window) if window else 0
            idx = torch.tensor(list(range(min(first, base), base)) + [base + j for j in range(n) if bits >> j & 1], dtype=torch.long)
            pages, offs = block_tables[b].long()[idx // page_size], idx % page_size
            for h in range(num_heads):
                K, V = k_cache[pages, h // group, offs, :].float(), v_cache[pages, h // group, offs, :].float()
                w = torch.softmax((K @ q[t, h * head_dim:(h + 1) * head_dim].float()) * scale, 0)
                out[t, h * head_dim:(h + 1) * head_dim] = (w @ V).to(out.dtype)


def logits_constrain(logits, owner=None, bias=None, history=None, penalties=None, windows=None, drafts=None, allowed=None,
                     allowed_rows=None, out=None):
    assert out is None
    for r in range(logits.shape[0]):
        q = r if owner is None else int(owner[r])
        if q >= 0:
            if bias is not None:
                for i in range(int(bias[0][q]), int(bias[0][q + 1])):
                    logits[r, int(bias[1][i])] += bias[2][i]
            said = history[1][int(history[0][q]):int(history[0][q + 1])].tolist()
            if drafts is not None:
                d0, d1 = int(drafts[0][q]), int(drafts[0][q + 1])
                said += [int(drafts[1][d0 + j]) for j in range(d1 - d0) if int(drafts[2][r]) >> j & 1]
            w = int(windows[q])
            said = said[-w:] if w else said
            rep, presence, frequency = penalties[q].tolist()
            for t in set(said):
                x = float(logits[r, t])
                if rep not in (0.0, 1.0):
                    x = x / rep if x > 0 else x * rep
                logits[r, t] = x - (presence + frequency * said.count(t))
        if allowed is not None and int(allowed_rows[r]) >= 0:
            words, token = allowed[int(allowed_rows[r])].long(), torch.arange(logits.shape[1])
            logits[r, words[token // 32] >> token % 32 & 1 == 0] = float("-inf")


def tree_accept(tokens, parents, chosen, q_start, path, counts, following):
    path.fill_(-1)
    for b in range(counts.shape[0]):
        a, n = int(q_start[b]), int(q_start[b + 1] - q_start[b])
        at, j = 0, 0
        while at is not None:
            path[a + j], j, last = at, j + 1, at
            at = next((i for i in range(at + 1, n) if parents[a + i] == at and tokens[a + i] == chosen[a + at]), None)
        counts[b], following[b] = j, chosen[a + last]


def tree_keep(tensors, slots, q_start, path, counts, axis=0):
    for t in tensors:
        old, ps, lead = t.clone(), t.shape[-2], (slice(None),) * axis
        inner = (slice(None),) * (t.dim() - axis - 3)
        for b in range(counts.shape[0]):
            a = int(q_start[b])
            for j in range(int(counts[b])):
                to, fro = int(slots[a + j]), int(slots[a + int(path[a + j])])
                t[lead + (to // ps,) + inner + (to % ps,)] = old[lead + (fro // ps,) + inner + (fro % ps,)]


def install(monkeypatch):
    from tgo_b200.kernels import ops
    emulated_beams.install(monkeypatch)
    for name in ("attention_tree", "logits_constrain", "tree_accept", "tree_keep"):
        monkeypatch.setattr(ops, name, globals()[name])


# ------------------------------------------------------------------------------ drafters


class Oracle:
    """Drafts that are right for `right` tokens, beside wrong ones: knows what every prompt's text will be."""

    def __init__(self, texts, right, wrong=2, vocab=10 ** 9):
        self.texts, self.right, self.wrong, self.vocab = texts, right, wrong, vocab

    def propose(self, tokens, nodes):
        tokens = list(tokens)
        text = next((t for t in self.texts if t[:len(tokens)] == tokens), [])
        drafted, parents, at = [], [], 0
        for t in text[len(tokens):len(tokens) + self.right]:
            for k in range(self.wrong):                    # wrong siblings first, one of them with a child
                drafted.append((t + 1 + k) % self.vocab)
                parents.append(at)
            if self.wrong:
                drafted.append(t)
                parents.append(len(drafted) - 1)
            drafted.append(t)
            parents.append(at)
            at = len(drafted)
        return drafted[:nodes], parents[:nodes]


class Noise:
    """Trees of any tokens."""

    def __init__(self, vocab, seed=0):
        import random
        self.vocab, self.rng = vocab, random.Random(seed)

    def propose(self, tokens, nodes):
        n = self.rng.randint(0, nodes)
        return [self.rng.randrange(self.vocab) for _ in range(n)], [self.rng.randint(0, i) for i in range(n)]
