"""Speculative greedy decoding: a draft engine proposes, the full engine checks a tree of proposals per pass.

A decoder pass over up to 16 tokens a window costs little more than one over a single token (the weights
and the encoder K/V are read once either way; beyond 16 the cross-attention reads them again), so every pass
of the full model checks a tree of tokens that a cheaper engine drafted: a model with the same vocabulary and far
fewer decoder layers, in bf16 or 4 bits (`WhisperEngine(decoder_format = 'mxfp4')`).  A step takes about as long per
layer in either, so the same model in 4 bits saves nothing as a draft (large-v3, one window, 64 tokens: 113 ms
without a draft, 138 ms with that one and every draft accepted).  Each round

* the draft decodes `draft_tokens` tokens greedily, noting its `draft_width` best candidates at each place;
* the full engine runs one `decode_tree` pass over the last accepted token and those candidates: the
  draft's first choices form the trunk, the other candidates are leaves beside it;
* from the root on, the full engine's own choice after a node selects the next node as long as it is
  among the candidates; its choice after the last accepted node is one more token;
* the accepted path joins both histories (`commit_tree`, `truncate_tree`), whose lengths then differ from
  window to window.

Every token is the full engine's argmax over its own history, so the ids are those of its greedy search;
a pass over several rows sums in another order than one over a single row, which can decide differently
between candidates whose scores agree to that rounding.  The reference has no counterpart.
"""
import numpy as np
import torch


def tree_layout(depth, width):
    """Parents [1 + depth * width] of the checked tree: node 0 is the last accepted token, nodes
    1 + d * width .. are the candidates of place d (the first one on the trunk)."""
    parents = [-1]
    for d in range(depth):
        trunk = 0 if d == 0 else 1 + (d - 1) * width
        parents += [trunk] * width
    return np.asarray(parents, dtype=np.int32)


def walk(choice, tokens, depth, width):
    """Accepted nodes (node 0 first) of one window: `choice` and `tokens` are the full engine's choice after
    and the token of every node."""
    path, node = [0], 0
    for d in range(depth):
        first = 1 + d * width
        hit = [first + j for j in range(width) if tokens[first + j] == choice[node]]
        if not hit:
            break
        node = hit[0]
        path.append(node)
        if node != first:                  # a leaf beside the trunk: nothing was drafted behind it
            break
    return path


def rows_per_window(engine, n):
    """Tokens of each of n windows that fit one pass of the engine."""
    return min(64, engine.max_batch * engine.max_beams * engine.max_prompt_len // n)


def feed(engine, lists, pad_token, reset=False):
    """Appends lists[i] (possibly empty) to the tree history of window i, in passes the engine has rows for;
    returns the logits [n, V] after each window's last token (zeros where there was none)."""
    n, most = len(lists), max(len(x) for x in lists)
    step = rows_per_window(engine, n)
    logits = None
    for at in range(0, most, step):
        part = [x[at: at + step] for x in lists]
        width = max(len(x) for x in part)
        tokens = np.full((n, width), pad_token, dtype=np.int32)        # shorter rows are padded behind
        for i, x in enumerate(part):
            tokens[i, :len(x)] = x
        z = engine.decode_tree(tokens, reset=reset and at == 0)
        engine.commit_tree([list(range(len(x))) for x in part])
        ends = [i for i, x in enumerate(lists) if at < len(x) <= at + step]
        if logits is None:
            logits = torch.zeros((n, z.shape[2]), dtype=z.dtype, device=z.device)
        if ends:
            logits[ends] = z[ends, [len(part[i]) - 1 for i in ends]]
    return logits


def generate(engine, draft, prompt, *, max_new_tokens, eos_token, pad_token, draft_tokens=4, draft_width=1,
             suppress=None, extras=None):
    """Greedy search of `engine` with `draft` proposing; same results layout as `WhisperEngine.generate`:
    tokens [B, steps], lengths [B], scores [B].  Both engines must hold the same encoded windows.
    `suppress`: token ids neither engine may choose.  `extras`: a dict that receives 'speculation', the
    number of passes of the full engine and of tokens they accepted."""
    prompt = np.ascontiguousarray(np.asarray(prompt, dtype=np.int32))
    if prompt.ndim == 1:
        prompt = prompt[None]
    n, s = prompt.shape
    steps, depth_max, width = int(max_new_tokens), int(draft_tokens), int(draft_width)
    if steps < 1 or s < 1:
        raise ValueError("prompt of %d tokens and %d new ones" % (s, steps))
    if depth_max < 1 or width < 1 or 1 + depth_max * width > 64:
        raise ValueError("a tree of %d x %d candidates: at least one, at most 63" % (depth_max, width))
    if draft is engine:
        raise ValueError("the draft must be another engine: both keep a history")
    if draft.dims["n_vocab"] != engine.dims["n_vocab"]:
        raise ValueError("draft and engine have vocabularies of %d and %d" % (draft.dims["n_vocab"], engine.dims["n_vocab"]))
    if engine._batch != n or draft._batch != n:
        raise ValueError("both engines must have encoded the %d windows of the prompt (they hold %d and %d)" % (
            n, engine._batch, draft._batch))
    for e in (engine, draft):
        if s + steps > e.max_text_len:
            raise ValueError("prompt %d + %d new tokens exceed the engine capacity (%d)" % (s, steps, e.max_text_len))
    rows = rows_per_window(engine, n)
    depth_max = min(depth_max, (rows - 1) // width)
    if depth_max < 1 or rows_per_window(draft, n) < 1:
        raise ValueError("%d rows per window and pass are too few for a tree: reserve a larger max_prompt_len" % rows)
    banned = None
    if suppress is not None:
        banned = torch.as_tensor(np.asarray(suppress, dtype=np.int64).reshape(-1), device=engine.device)

    def keep(logits):
        return logits if banned is None else logits.index_fill(logits.dim() - 1, banned.to(logits.device), float("-inf"))

    logits = keep(feed(engine, prompt.tolist(), pad_token, reset=True))
    first = logits.argmax(dim=-1)
    gain = torch.log_softmax(logits, dim=-1).gather(1, first[:, None])[:, 0].tolist()
    feed(draft, prompt.tolist(), pad_token, reset=True)
    out = [[int(t)] for t in first.tolist()]
    scores = [float(g) for g in gain]
    lacking = [[] for _ in range(n)]        # accepted tokens the draft has not seen, the last one excepted
    passes = accepted = 0

    def done(i):
        return out[i][-1] == eos_token or len(out[i]) >= steps

    ended = set()
    while True:
        # windows that have ended give their positions back
        over = [i for i in range(n) if done(i) and i not in ended]
        if over:
            ended.update(over)
            for e in (engine, draft):
                left = e.tree_lengths()
                left[over] = 0
                e.truncate_tree(left)
        live = [i for i in range(n) if i not in ended]
        if not live:
            break
        draft_len = draft.tree_lengths()
        fed = [lacking[i] + [out[i][-1]] if i in live else [] for i in range(n)]
        room = engine.max_text_len - int(engine.tree_lengths().max())
        draft_room = min(draft.max_text_len - int(draft_len[i]) - len(fed[i]) for i in live)
        depth = max(0, min(depth_max, (room - 1) // width, draft_room + 1, max(steps - len(out[i]) for i in live) - 1))
        tokens = np.full((n, 1 + depth * width), pad_token, dtype=np.int32)
        tokens[live, 0] = [out[i][-1] for i in live]
        if depth > 0:
            z = feed(draft, fed, pad_token)
            for d in range(depth):
                best = torch.topk(keep(z), width, dim=-1).indices.cpu().numpy()
                tokens[:, 1 + d * width: 1 + (d + 1) * width] = best
                if d + 1 < depth:
                    z = feed(draft, [[int(best[i, 0])] if i in live else [] for i in range(n)], pad_token)
        z = keep(engine.decode_tree(tokens, np.tile(tree_layout(depth, width)[None], (n, 1))))
        choice_t = z.argmax(dim=-1)
        gains = (z.gather(2, choice_t[..., None])[..., 0] - torch.logsumexp(z, dim=-1)).cpu().numpy()
        choice = choice_t.cpu().numpy()
        passes += 1
        commits, lengths = [[] for _ in range(n)], draft_len.copy()
        for i in live:
            path, kept = walk(choice[i], tokens[i], depth, width), 0
            for a in path:                           # what the full engine says after each accepted node
                scores[i] += float(gains[i][a])
                out[i].append(int(choice[i][a]))
                kept += 1
                if done(i):
                    break
            accepted += kept
            path = commits[i] = path[:kept]
            if depth > 0:
                # the draft holds the trunk up to the last token but one; a leaf is not on it
                trunk = sum(1 for k, a in enumerate(path) if k and a == 1 + (k - 1) * width)
                have = min(trunk, depth - 1)
                lengths[i] += len(fed[i]) + have
                lacking[i] = [int(tokens[i][a]) for a in path[1 + have:]]
            else:
                lacking[i] = fed[i]
        engine.commit_tree(commits)
        if depth > 0:
            draft.truncate_tree(lengths)
    tokens = np.full((n, steps), pad_token, dtype=np.int32)
    lens = np.zeros(n, np.int32)
    for i in range(n):
        tokens[i, :len(out[i])] = out[i]
        lens[i] = len(out[i]) - (1 if out[i][-1] == eos_token else 0)
    if extras is not None:
        extras["speculation"] = {"passes": passes, "tokens": accepted}
    return tokens, lens, np.asarray(scores, dtype=np.float32)
