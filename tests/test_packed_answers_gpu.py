"""Packed answers (models/qwen_answers.py) against the fp32 model run on each request's whole sequence:
questions of different lengths about one image, then token by token; the same without an image."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _setup(precision="bf16", seed=4):
    from appcorr_b200.models.qwen25vl import PRESETS, Qwen25VL
    from appcorr_b200.models.qwen_engine import QwenVLEngine

    cfg = PRESETS["tiny"]
    m = Qwen25VL(cfg).init_weights(seed).to(DEV).eval()
    return cfg, m, QwenVLEngine(m, DEV, precision)


def _oracle(m, x, pos):
    from appcorr_b200.models.qwen25vl import mrope_tables

    sin, cos = (v.to(DEV) for v in mrope_tables(m.cfg, pos.cpu()))
    with torch.no_grad():
        for i, ly in enumerate(m.layers):
            x = ly.approx(x, sin, cos, {}, f"l{i}")
        return m.lm_head(m.norm(x[-1:]))[0]


def _rel(a, b):
    return ((a.float() - b.float()).norm() / b.float().norm()).item()


@pytest.mark.parametrize("precision,tol", [("bf16", 3e-2), ("fp8", 0.15)])
def test_questions_about_one_image(precision, tol):
    """The tolerances are those of the engine's own prefill tests at these precisions."""
    from appcorr_b200.models.qwen25vl import mrope_positions
    from appcorr_b200.models.qwen_answers import PackedAnswers
    from appcorr_b200.ops.native import check_errors

    cfg, m, eng = _setup(precision)
    g = torch.Generator().manual_seed(7)
    nb, na = 8, 70  # a prompt that ends inside its second page
    ids = torch.randint(0, cfg.vocab, (nb + na,), generator=g).to(DEV)
    img = torch.randint(0, 256, (1, 224, 224, 3), dtype=torch.uint8, device=DEV)
    sess = eng.new_session(224, 224, nb, na)
    eng.vision(sess, img)
    eng.embed_text(sess, ids)
    eng.approx(sess)
    pa = PackedAnswers(eng, max_requests=5, max_own=300, max_step=400, session=sess)
    q = [torch.randint(0, cfg.vocab, (n,), generator=g).to(device=DEV, dtype=torch.int32) for n in (1, 130, 17, 126)]
    with torch.no_grad():
        prompt = m.embed(ids[:nb], m.visual(img[0]), ids[nb:])
    pos0 = mrope_positions(nb, 8, 8, na)
    seqs = [x.long() for x in q]
    step_ids, lens = torch.cat(q), torch.tensor([x.numel() for x in q], dtype=torch.int32, device=DEV)
    for _ in range(4):  # the questions, then three tokens: the fourth request crosses into its second page
        logits = pa.step(step_ids, lens).clone()
        torch.cuda.synchronize()
        check_errors(torch.device(DEV))
        for b, s in enumerate(seqs):
            after = int(pos0.max()) + 1 + torch.arange(s.numel())
            pos = torch.cat([pos0, after.expand(3, -1)], 1)
            want = _oracle(m, torch.cat([prompt, m.embed_tokens(s)]), pos)
            assert _rel(logits[b], want) < tol, b
        step_ids = logits.argmax(1).to(torch.int32)  # both sides go on with the engine's token
        seqs = [torch.cat([s, step_ids[b:b + 1].long()]) for b, s in enumerate(seqs)]
        lens = torch.ones_like(lens)
    assert pa.pages_missing == 0


def test_requests_without_an_image_and_generate():
    from appcorr_b200.models.qwen_answers import PackedAnswers

    cfg, m, eng = _setup(seed=5)
    g = torch.Generator().manual_seed(9)
    q = [torch.randint(0, cfg.vocab, (n,), generator=g).to(device=DEV, dtype=torch.int32) for n in (40, 3, 150)]
    pa = PackedAnswers(eng, max_requests=3, max_own=200, max_step=256)
    logits = pa.step(torch.cat(q), torch.tensor([40, 3, 150], dtype=torch.int32, device=DEV)).clone()
    for b, s in enumerate(q):
        want = _oracle(m, m.embed_tokens(s.long()), torch.arange(s.numel()).expand(3, -1))
        assert _rel(logits[b], want) < 3e-2, b
    out = pa.generate(q, 5)
    assert out.shape == (3, 5) and torch.equal(out[:, 0], logits.argmax(1).to(torch.int32))
    assert torch.equal(out, pa.generate(q, 5))  # the same bits again


def test_refusals():
    from appcorr_b200.models.qwen_answers import PackedAnswers

    cfg, m, eng = _setup()
    with pytest.raises(ValueError):
        PackedAnswers(eng, 2, 100, 64, session=eng.new_session(224, 224, 4, 4))  # its prompt was not run
    pa = PackedAnswers(eng, max_requests=2, max_own=100, max_step=64)
    tok = torch.zeros(65, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError):
        pa.step(tok, torch.tensor([65], dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError):
        pa.generate([tok[:3], tok[:0]], 1)
    with pytest.raises(RuntimeError):
        pa.generate([tok[:60]], 70)  # 129 tokens in one page
    torch.cuda.synchronize()
