"""TreeDecoder on the GPU: its logits against the model runner's own decoding,
byte for byte; trees against the paths that they hold; greedy decoding with
drafts against greedy decoding without."""
import numpy as np
import pytest
import torch

from i_whisper_b200.checkpoint import ModelDims, synthetic_state_dict
from i_whisper_b200.synthetic import synthetic_mel_batch

pytestmark = pytest.mark.gpu

DIMS = ModelDims(80, 1500, 384, 6, 1, 51865, 448, 384, 6, 2)


@pytest.fixture(scope="module")
def setup():
    from i_whisper_b200.model import WhisperIntB200
    sd = synthetic_state_dict(DIMS, 3)
    mel = torch.from_numpy(synthetic_mel_batch(DIMS.n_mels, [5, 6, 7], float(sd["encoder.input_alpha"][0]))).cuda()
    model = WhisperIntB200(DIMS, sd)
    return sd, model, model.encoder(mel).clone()


def dense_logits(model, xa, tokens):
    """[len(tokens), n_vocab]: logits after each token, one token at a time through the runner's dense cache."""
    ws = model._dec_workspace(1, len(tokens) + 1)
    ws["tokens"].zero_()
    ws["state"].zero_()
    ws["state"][:, 3] = -1
    ws["pos"].zero_()
    ws["tk"].fill_(1)
    ws["step"].fill_(3)
    model.cross_kv(xa[None].contiguous(), None, ws)
    t = torch.tensor(tokens, dtype=torch.int64, device="cuda")
    out = []
    for i in range(len(tokens)):
        ws["step"].fill_(3)
        model._dec_forward(ws, 1, 1, t[i:].data_ptr(), 1, i, graph_mode=False)
        out.append(ws["logits"][0, :DIMS.n_vocab].clone())
    return torch.stack(out)


def random_tree(rng, n, vocab=51865):
    return rng.integers(0, vocab, n).tolist(), [-1] + [int(rng.integers(-1, i)) for i in range(1, n)]


def test_chains_match_the_dense_decoder(setup):
    from i_whisper_b200.tree import TreeDecoder
    _, model, xa = setup
    rng = np.random.default_rng(0)
    toks = [rng.integers(0, DIMS.n_vocab, n).tolist() for n in (19, 1, 7)]
    dec = TreeDecoder(model, xa)
    got = dec.step(toks, top=3)
    want = torch.cat([dense_logits(model, xa[b], toks[b]) for b in range(3)])
    assert torch.equal(got.logits, want)
    # the scores are those logits'
    lp = torch.log_softmax(want.double() / model.logit_alpha, 1)
    assert torch.allclose(got.top_logprobs.double(), torch.gather(lp, 1, got.top_ids), atol=1e-4)
    # the second part of the context in another pass
    dec.accept([range(n) for n in (19, 1, 7)])
    more = [rng.integers(0, DIMS.n_vocab, n).tolist() for n in (2, 30, 0)]
    got = dec.step(more)
    want = [dense_logits(model, xa[b], toks[b] + more[b])[len(toks[b]):] for b in range(3) if more[b]]
    assert torch.equal(got.logits, torch.cat(want))


def test_tree_nodes_match_their_paths(setup):
    from i_whisper_b200.tree import TreeDecoder
    _, model, xa = setup
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, DIMS.n_vocab, n).tolist() for n in (5, 17, 30)]
    dec = TreeDecoder(model, xa, page_size=8)
    dec.step(prompts)
    dec.accept([range(len(p)) for p in prompts])
    trees = [random_tree(rng, n) for n in (40, 9, 1)]
    got = dec.step([t for t, _ in trees], [p for _, p in trees]).logits
    start, paths = 0, []
    for b, (t, p) in enumerate(trees):
        node = int(rng.integers(0, len(t)))
        path = [node]
        while p[path[0]] >= 0:
            path.insert(0, p[path[0]])
        want = dense_logits(model, xa[b], prompts[b] + [t[i] for i in path])[len(prompts[b]):]
        assert torch.equal(got[[start + i for i in path]], want)
        start += len(t)
        paths.append(path)
    # accepting a path leaves the cache as decoding it would have
    dec.accept(paths)
    nxt = [[11], [12], [13]]
    got = dec.step(nxt).logits
    for b, (t, _) in enumerate(trees):
        assert torch.equal(got[b], dense_logits(model, xa[b], prompts[b] + [t[i] for i in paths[b]] + nxt[b])[-1])


def test_greedy_is_the_same_with_any_drafts(setup):
    from i_whisper_b200 import _lib
    from i_whisper_b200.tree import TreeDecoder
    _, model, xa = setup
    sot = model.tokens_spec["sot_sequence"]
    prompts, n = [list(sot), list(sot) + [400, 11], list(sot)[:1]], 24
    dec = TreeDecoder(model, xa)
    plain = dec.greedy(prompts, n, lambda b, h: ([], []))
    assert dec.passes == n - 1 and all(len(o) == n for o in plain)
    rng = np.random.default_rng(2)

    def oracle_and_noise(b, hist):
        """The right continuation hidden in a tree of wrong ones (sometimes cut short)."""
        done = len(hist) - len(prompts[b])
        right = plain[b][done:done + int(rng.integers(0, 5))]
        t, p, last = [], [], -1
        for tok in right:
            for _ in range(int(rng.integers(0, 3))):
                t.append(int(rng.integers(0, DIMS.n_vocab)))
                p.append(int(rng.integers(-1, len(t) - 1)) if len(t) > 1 else -1)
            t.append(tok)
            p.append(last)
            last = len(t) - 1
        return t, p

    drafted = TreeDecoder(model, xa, page_size=8)
    assert drafted.greedy(prompts, n, oracle_and_noise) == plain
    assert drafted.passes < n - 1
    # the pool holds exactly the contexts' pages
    used = sum(-(-c // 8) for c in drafted.lens)
    assert int(drafted.head.item()) == used
    owned = drafted.table[drafted.table >= 0].tolist() + drafted.free[used:].tolist()
    assert sorted(owned) == list(range(drafted.free.numel()))
    assert _lib.device_status(clear=True) == 0


def test_zero_point_form(setup):
    from i_whisper_b200.model import WhisperIntB200
    from i_whisper_b200.tree import TreeDecoder
    sd, model, xa = setup
    unfolded = WhisperIntB200(DIMS, sd, fold_zero_points=False)
    rs = torch.empty(xa.shape[0] * xa.shape[1], dtype=torch.int32, device="cuda")
    from i_whisper_b200 import _lib
    _lib.call("iw_rowsum_i8", xa.data_ptr(), xa.shape[2], rs.numel(), xa.shape[2], rs.data_ptr(),
              torch.cuda.current_stream().cuda_stream)
    toks = [[1, 2, 3], [4], [5, 6]]
    a, b = TreeDecoder(model, xa).step(toks), TreeDecoder(unfolded, xa, rs).step(toks)
    assert torch.equal(a.logits, b.logits)


def test_refusals(setup):
    from i_whisper_b200.tree import TreeDecoder
    _, model, xa = setup
    dec = TreeDecoder(model, xa, pages=4)
    with pytest.raises(RuntimeError, match="3 lists"):
        dec.step([[1]])
    with pytest.raises(RuntimeError, match="no tokens"):
        dec.step([[], [], []])
    with pytest.raises(RuntimeError, match="448"):
        dec.step([[1] * 449, [], []])
    with pytest.raises(RuntimeError, match="out of cache pages"):
        dec.step([[1] * 40, [1] * 40, [1]])
    with pytest.raises(RuntimeError, match="parents"):
        dec.step([[1], [1], []], [[-1], [], []])
    dec.step([[1, 2], [], [3]])
    with pytest.raises(RuntimeError, match="increasing"):
        dec.accept([[1, 0], [], []])
    with pytest.raises(RuntimeError, match="features"):
        TreeDecoder(model, xa[0])


def test_features_of_any_strides(setup):
    """Rows taken out of a batch and one utterance decoded several times, as of contiguous copies."""
    from i_whisper_b200.tree import TreeDecoder
    _, model, xa = setup
    for some in (xa[::2], xa[1:2].expand(3, -1, -1), xa.flip(0), xa.transpose(1, 2).contiguous().transpose(1, 2)):
        toks = [[1, 2, 3], [4], [5, 6]][:len(some)]
        want = [dense_logits(model, x, t) for x, t in zip(some, toks)]
        assert torch.equal(TreeDecoder(model, some).step(toks).logits, torch.cat(want))


def test_features_refusals(setup):
    from i_whisper_b200.model import WhisperIntB200
    from i_whisper_b200.tree import TreeDecoder
    sd, model, xa = setup
    unfolded = WhisperIntB200(DIMS, sd, fold_zero_points=False)
    rs = torch.zeros(xa.shape[0] * xa.shape[1], dtype=torch.int32, device="cuda")
    for m, x, r, match in ((model, xa.cpu(), None, "features"), (unfolded, xa, None, "rs_xa"), (unfolded, xa, rs[1:], "rs_xa"),
                           (unfolded, xa, rs.long(), "rs_xa"), (unfolded, xa, rs.cpu(), "rs_xa"),
                           (unfolded, xa, rs.repeat(2)[::2], "rs_xa")):
        with pytest.raises(RuntimeError, match=match):
            TreeDecoder(m, x, r)
    with pytest.raises(RuntimeError, match="contiguous"):  # the runner's own decoding takes no strides
        model.decode(xa[::2], None, 4)


def test_a_refused_pass_leaves_the_pool_as_it_was(setup):
    from i_whisper_b200.tree import TreeDecoder
    _, model, xa = setup
    dec = TreeDecoder(model, xa, pages=4)
    with pytest.raises(RuntimeError, match="pass"):
        dec.accept([[], [], []])
    dec.step([[1, 2, 3], [4], []])
    dec.accept([[0, 1, 2], [0], []])
    for refused in (lambda: dec.step([[1] * 40, [1] * 40, [1]]), lambda: dec.step([[1], [1], [1]], top=33)):
        with pytest.raises(RuntimeError, match="out of cache pages|top"):
            refused()
        with pytest.raises(RuntimeError, match="pass"):
            dec.accept([[], [], []])
        assert dec.head.item() == 2 and dec.lens == [3, 1, 0]
    got = dec.step([[5], [], [6] * 20]).logits  # the two pages that are left
    assert torch.equal(got[0], dense_logits(model, xa[0], [1, 2, 3, 5])[-1])
    assert torch.equal(got[1:], dense_logits(model, xa[2], [6] * 20))
    dec.accept([[0], [], [0]])
    owned = dec.table[:, 0].tolist() + dec.free[3:].tolist()
    assert dec.head.item() == 3 and sorted(owned) == [0, 1, 2, 3]


def test_accept_takes_a_path_of_every_utterance(setup):
    from i_whisper_b200.tree import TreeDecoder
    _, model, xa = setup
    dec = TreeDecoder(model, xa)
    dec.step([[1, 2], [4], [3]])
    for paths in ([[0, 1]], [[0, 1], [0]], [[0, 1], [0], [0], [0]]):
        with pytest.raises(RuntimeError, match="3 paths"):
            dec.accept(paths)
    dec.accept([[0, 1], [0], []])
    assert dec.lens == [2, 1, 0] and dec.ctx.tolist() == [2, 1, 0]
    with pytest.raises(RuntimeError, match="pass"):
        dec.accept([[0, 1], [0], []])


def test_accept_takes_only_branches(setup):
    from i_whisper_b200.tree import TreeDecoder
    _, model, xa = setup
    dec = TreeDecoder(model, xa)
    # 0 and 1 follow the context, 2 and 3 follow 0, 4 follows 1; 5's parent is no earlier token
    dec.step([[1, 2, 3, 4, 5, 6], [1, 2, 3], []], [[-1, -1, 0, 0, 1, 7], [-1, 0, 1], []])
    for paths in ([[0, 1], [], []], [[2], [], []], [[0, 2, 3], [], []], [[0, 4], [], []], [[0, 5], [], []],
                  [[], [1], []], [[], [0, 2], []]):
        with pytest.raises(RuntimeError, match="branch"):
            dec.accept(paths)
    assert dec.lens == [0, 0, 0]
    dec.accept([[5], [0, 1], []])
    assert dec.lens == [1, 2, 0]
    dec.step([[1, 2, 3], [1], []])  # chains
    for paths in ([[1, 2], [], []], [[0, 2], [], []]):
        with pytest.raises(RuntimeError, match="branch"):
            dec.accept(paths)
    dec.accept([[0, 1], [0], []])
    assert dec.lens == [3, 3, 0]


def test_token_ids_outside_the_vocabulary(setup):
    from i_whisper_b200.tree import TreeDecoder
    _, model, xa = setup
    dec = TreeDecoder(model, xa)
    for bad in (-1, DIMS.n_vocab, 2 ** 40):
        with pytest.raises(RuntimeError, match="token ids"):
            dec.step([[1, 2], [], [3, bad]])
        with pytest.raises(RuntimeError, match="token ids"):
            dec.step([[1, bad], [], [3]], [[-1, 0], [], [-1]])
    last = DIMS.n_vocab - 1
    assert torch.equal(dec.step([[0, last], [], []]).logits, dense_logits(model, xa[0], [0, last]))


def test_greedy_needs_prompts(setup):
    from i_whisper_b200.tree import TreeDecoder
    _, model, xa = setup
    for prompts in ([[], [1], [2]], [[1], [], [2]], [[], [], []]):
        with pytest.raises(RuntimeError, match="prompt"):
            TreeDecoder(model, xa).greedy(prompts, 4, lambda b, h: ([], []))
