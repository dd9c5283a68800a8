"""Packed answers (models/qwen_answers.py) at the edges of a step: requests that bring no token, lengths and
ids that do not fit together, errors. The oracle and its tolerance are those of
test_packed_answers_gpu.py."""
import pytest
import torch

from test_packed_answers_gpu import DEV, _oracle, _rel, _setup

pytestmark = pytest.mark.gpu


def _ints(*values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


class Batch:
    """Requests without an image, with their sequences beside them."""

    def __init__(self, lengths, seed=5, **kw):
        from appcorr_b200.models.qwen_answers import PackedAnswers

        self.cfg, self.m, eng = _setup(seed=seed)
        self.g = torch.Generator().manual_seed(seed + 4)
        self.seqs = [torch.empty(0, dtype=torch.long, device=DEV) for _ in lengths]
        self.pa = PackedAnswers(eng, **(dict(max_requests=len(lengths), max_own=200, max_step=256) | kw))
        self.first = self.step(*lengths)

    def step(self, *lengths):
        new = [torch.randint(0, self.cfg.vocab, (n,), generator=self.g).to(DEV) for n in lengths]
        out = self.pa.step(torch.cat(new).to(torch.int32), _ints(*lengths)).clone()
        self.seqs = [torch.cat([s, x]) for s, x in zip(self.seqs, new)]
        return out

    def check(self, logits, b):
        from appcorr_b200.ops.native import check_errors

        torch.cuda.synchronize()
        check_errors(torch.device(DEV))
        s = self.seqs[b]
        want = _oracle(self.m, self.m.embed_tokens(s), torch.arange(s.numel()).expand(3, -1))
        assert _rel(logits[b], want) < 3e-2, b


@pytest.mark.parametrize("idle", [(0,), (1,), (2,), (0, 1), (1, 2), (0, 2)])
def test_requests_that_bring_no_token(idle):
    """Their logits stay, the others go on, and they can go on later."""
    t = Batch((40, 3, 150))
    last = t.first
    for n in (1, 2):
        out = t.step(*(0 if b in idle else n for b in range(3)))
        for b in range(3):
            if b in idle:
                assert torch.equal(out[b], last[b]), b
            else:
                t.check(out, b)
    out = t.step(1, 1, 1)
    for b in range(3):
        t.check(out, b)


def test_step_of_no_tokens_at_all():
    t = Batch((40, 3, 150))
    assert torch.equal(t.step(0, 0, 0), t.first)
    out = t.step(2, 0, 1)
    t.check(out, 0)
    assert torch.equal(out[1], t.first[1])
    assert t.pa.step(_ints(), _ints()).shape == (0, t.cfg.vocab)


def test_request_that_has_not_begun():
    """Zeros before its first token, also when the batch was used before."""
    t = Batch((5, 0, 9))
    assert bool((t.first[1] == 0).all())
    t.check(t.first, 0)
    t.check(t.first, 2)
    t.step(1, 4, 0)
    t.pa.reset()
    assert bool((t.pa.step(_ints(3), _ints(1, 0, 0))[1:] == 0).all())


def test_lengths_and_ids_that_do_not_fit():
    """Tokens that ids does not hold are not taken, and counted; ids past the lengths are padding."""
    t = Batch((40, 3, 150))
    ids = torch.randint(0, t.cfg.vocab, (7,), generator=t.g).to(device=DEV, dtype=torch.int32)
    for lengths, taken in (((2, 9, 4), (2, 5, 0)), ((7, 1, 1), (7, 0, 0)), ((1 << 30, 1 << 30, 1 << 30), (7, 0, 0)), ((1, 2, 1), (1, 2, 1)),
                           ((-3, 2, 5), (0, 2, 5))):
        missing = t.pa.tokens_missing
        out = t.pa.step(ids, _ints(*lengths)).clone()
        at = 0
        for b, n in enumerate(taken):
            t.seqs[b] = torch.cat([t.seqs[b], ids[at:at + n].long()])
            at += n
            t.check(out, b)
        assert t.pa.tokens_missing - missing == max(sum(max(n, 0) for n in lengths) - 7, 0)
        assert t.pa.held.tolist() == [s.numel() for s in t.seqs]
    assert t.pa.pages_missing == 0
    assert t.pa.step(_ints(), _ints(0, 2, 0)).shape[0] == 3 and t.pa.held.tolist() == [s.numel() for s in t.seqs]


def test_ids_that_are_no_rows_of_the_embedding_are_refused():
    """On the host, of another type or stride, outside the vocabulary: nothing runs, nothing is forgotten."""
    t = Batch((40, 3, 150))
    one, vocab = _ints(1, 1, 1), t.cfg.vocab
    for ids, q_len in ((_ints(1, 2, 3).cpu(), one), (_ints(1, 2, 3).long(), one), (_ints(1, 9, 2, 9, 3, 9)[::2], one),
                       (_ints(1, 2, 3), one.cpu()), (_ints(1, 2, 3), one.long()), (_ints(1, 2, 3), one[None])):
        with pytest.raises(ValueError, match="must be int32"):
            t.pa.step(ids, q_len)
    for ids in (_ints(1, vocab), _ints(-1, 1), torch.tensor([vocab]), torch.tensor([(1 << 32) + 5])):
        with pytest.raises(ValueError, match="vocabulary"):
            t.pa.generate([_ints(1), ids], 2)
    assert t.pa.held.tolist() == [40, 3, 150]
    out = t.pa.step(_ints(1, 2, 3)[None], _ints(1, 9, 1, 9, 1, 9)[::2])  # shapes that make no difference
    t.seqs[1] = torch.cat([t.seqs[1], _ints(2).long()])
    t.check(out, 1)


def test_generate_raises_recorded_errors():
    from appcorr_b200.ops.native import err_word

    t = Batch((4, 3))
    questions = [_ints(1, 2), _ints(3)]
    want, step, calls = t.pa.generate(questions, 3), t.pa.step, []

    def last_step_fails(ids, q_len):
        out = step(ids, q_len)
        calls.append(1)
        if len(calls) == 3:
            err_word(torch.device(DEV)).fill_(3)
        return out

    t.pa.step = last_step_fails
    with pytest.raises(RuntimeError, match="epilogue wait timed out"):
        t.pa.generate(questions, 3)
    t.pa.step = step
    assert torch.equal(t.pa.generate(questions, 3), want)


def test_generate_no_tokens():
    t = Batch((4, 3))
    out = t.pa.generate([_ints(1, 2), _ints(3)], 0)
    assert out.shape == (2, 0) and out.dtype == torch.int32 and out.device == t.pa.held.device
    with pytest.raises(ValueError, match="-1 tokens"):
        t.pa.generate([_ints(1)], -1)
