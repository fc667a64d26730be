"""generate(repetition_penalty, presence_penalty, frequency_penalty, logit_bias): the chosen tokens and processed logits against the same model's raw logits under the
same history (teacher forcing), processed by transformers' own class and by plain arithmetic in 64 bits."""
import math

import pytest
import torch

from conftest import load_golden

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def case():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from modelcompose_amd.model.builder import build_from_state_dict
    a, meta, sd = load_golden("g4_e2e_vision")
    return build_from_state_dict(meta, sd), a["input_ids"].cuda(), {"vision": a["pixels"].cuda()}


def _raw(model, ids, modal, new):
    """The unprocessed logits of every step when the model is fed `new`."""
    _, lg = model.generate(ids, modal_inputs=modal, max_new_tokens=new.shape[1], ignore_eos=True, forced_ids=new, return_step_logits=True)
    return lg.cpu()


def _processed(raw, prompt, new, rep, pres, freq, bias):
    V = raw.shape[-1]
    out = raw.double().clone()
    for b in range(raw.shape[0]):
        for s in range(raw.shape[1]):
            gen = new[b, :s].tolist()
            for t in {t for t in prompt[b].tolist() + gen if 0 <= t < V}:
                x = out[b, s, t]
                out[b, s, t] = x / rep if x > 0 else x * rep
            for t in set(gen):
                out[b, s, t] -= freq * gen.count(t) + pres
            for t, v in bias.items():
                out[b, s, t] += v
    return out


@pytest.mark.parametrize("rep,pres,freq,bias", [(1.7, 0.0, 0.0, {}), (0.6, 0.0, 0.0, {}), (1.0, 0.8, 0.5, {}), (1.3, -0.4, 0.9, {3: 2.5, 17: -math.inf, 60: -1.0})])
def test_chosen_tokens_and_scores(case, rep, pres, freq, bias):
    model, ids, modal = case
    n = 9
    res, got = model.generate(ids, modal_inputs=modal, max_new_tokens=n, ignore_eos=True, return_step_logits=True, repetition_penalty=rep, presence_penalty=pres,
                              frequency_penalty=freq, logit_bias=bias)
    new = res[:, ids.shape[1]:]
    raw = _raw(model, ids, modal, new)
    want = _processed(raw, ids.cpu(), new.cpu(), rep, pres, freq, bias)
    got = got.cpu().double()
    assert torch.equal(torch.isinf(got), torch.isinf(want))
    fin = torch.isfinite(want)
    # at most four fp32 roundings of numbers no larger than the logit before and after and what is added
    mag = raw.double().abs() * max(rep, 1 / rep) + want.abs().nan_to_num(posinf=0.0) + 3 * (abs(pres) + n * abs(freq) + 2.5)
    assert ((got - want).abs() <= 4 * 2.0 ** -24 * mag)[fin].all()
    assert torch.equal(new.cpu(), got.argmax(-1))
    if bias:
        assert not (new == 17).any()


def test_repetition_penalty_is_transformers_own(case):
    from transformers.generation.logits_process import RepetitionPenaltyLogitsProcessor
    model, ids, modal = case
    res, got = model.generate(ids, modal_inputs=modal, max_new_tokens=6, ignore_eos=True, return_step_logits=True, repetition_penalty=1.4)
    new = res[:, ids.shape[1]:].cpu()
    raw = _raw(model, ids, modal, new.cuda())
    proc = RepetitionPenaltyLogitsProcessor(1.4)
    for b in range(len(new)):
        text = ids[b].cpu()
        text = text[(text >= 0) & (text < raw.shape[-1])]                     # (the class has no answer for the sentinels of the modal tokens)
        for s in range(new.shape[1]):
            want = proc(torch.cat([text, new[b, :s]])[None], raw[b, s][None].clone())
            assert torch.allclose(got[b, s].cpu(), want[0], rtol=1e-6, atol=0)


def test_neutral_values_change_nothing_and_sampling_combines(case):
    model, ids, modal = case
    plain = model.generate(ids, modal_inputs=modal, max_new_tokens=7, ignore_eos=True)
    kw = dict(modal_inputs=modal, max_new_tokens=7, ignore_eos=True)
    assert torch.equal(plain, model.generate(ids, repetition_penalty=1.0, presence_penalty=0.0, frequency_penalty=0.0, logit_bias={}, **kw))
    assert torch.equal(plain, model.generate(ids, logit_bias={5: 0.0}, **kw))                    # the per-token path, nothing changed
    greedy = model.generate(ids, repetition_penalty=1.5, **kw)
    assert torch.equal(greedy, model.generate(ids, repetition_penalty=1.5, do_sample=True, top_k=1, temperature=0.7, **kw))
    a, b = (model.generate(ids, repetition_penalty=1.5, do_sample=True, temperature=1.5, seed=4, **kw) for _ in range(2))
    assert torch.equal(a, b)
    forced = model.generate(ids, logit_bias={42: 1e4}, **kw)
    assert (forced[:, ids.shape[1]:] == 42).all()
    assert torch.equal(plain, model.generate(ids, **kw))                                        # and nothing stays behind


def test_hooks_and_end_of_sequence(case):
    model, ids, modal = case
    eos = model.config.eos_token_id
    kw = dict(modal_inputs=modal, max_new_tokens=40)
    res = model.generate(ids, logit_bias={eos: 1e4}, **kw)
    assert res.shape[1] == ids.shape[1] + 1 and (res[:, -1] == eos).all()
    seen = []
    res = model.generate(ids, logit_bias={eos: -math.inf}, repetition_penalty=1.2, stopping_criteria=[lambda s, _: seen.append(s.shape[1]) or s.shape[1] >= ids.shape[1] + 4], **kw)
    assert res.shape[1] == ids.shape[1] + 4 and seen == [ids.shape[1] + i for i in (1, 2, 3, 4)]


def test_refusals(case):
    model, ids, modal = case
    V = model.config.vocab_size
    for bad in (dict(repetition_penalty=0.0), dict(repetition_penalty=-1.0), dict(repetition_penalty=math.inf), dict(presence_penalty=math.nan), dict(frequency_penalty=math.inf),
                dict(logit_bias={V: 1.0}), dict(logit_bias={-1: 1.0}), dict(logit_bias={1: math.nan})):
        with pytest.raises(ValueError):
            model.generate(ids, modal_inputs=modal, max_new_tokens=2, **bad)
    with pytest.raises(NotImplementedError):
        model.generate(ids, modal_inputs=modal, max_new_tokens=2, num_beams=2, repetition_penalty=1.2)
    with pytest.raises(ValueError):
        model.generate(ids, modal_inputs=modal, max_new_tokens=2, ignore_eos=True, forced_ids=torch.zeros(len(ids), 2, dtype=torch.int64), presence_penalty=1.0)


class _Recorder:
    def __init__(self):
        self.got, self.ended = [], False

    def put(self, t):
        self.got.append(t)

    def end(self):
        self.ended = True


@pytest.mark.parametrize("kw", [dict(presence_penalty=1e4), dict(presence_penalty=1e4, do_sample=True, temperature=1.3, seed=3), dict(repetition_penalty=1.1, presence_penalty=1e4)])
@pytest.mark.parametrize("last", [0, 1, 4, 17])
def test_nothing_is_streamed_after_the_end(case, kw, last, monkeypatch):
    """A streamer and the criteria see the answer and nothing behind it.  The presence penalty makes the tokens of a row distinct, so that any of them can be
    declared the end of the sequence."""
    model, ids, modal = case
    one, pix = ids[:1], {"vision": modal["vision"][:1]}
    free = model.generate(one, modal_inputs=pix, max_new_tokens=30, ignore_eos=True, **kw)[:, one.shape[1]:]
    assert free[0].unique().numel() == 30
    monkeypatch.setattr(model.config, "eos_token_id", int(free[0, last]))
    rec, lengths = _Recorder(), []
    res = model.generate(one, modal_inputs=pix, max_new_tokens=30, streamer=rec, stopping_criteria=[lambda s, _: bool(lengths.append(s.shape[1]))], **kw)
    assert torch.equal(res[:, one.shape[1]:], free[:, :last + 1])
    assert rec.ended and torch.equal(torch.stack(rec.got[1:], 1), free[:, :last + 1].cpu())
    assert lengths == [one.shape[1] + i + 1 for i in range(last + 1)]
    assert torch.equal(res, model.generate(one, modal_inputs=pix, max_new_tokens=30, **kw))            # and the loop without hooks


def test_streaming_goes_on_until_every_row_has_ended(case):
    model, ids, modal = case
    eos = model.config.eos_token_id
    rec = _Recorder()
    res = model.generate(ids, modal_inputs=modal, max_new_tokens=20, streamer=rec, logit_bias={eos: 1e4})
    assert res.shape[1] == ids.shape[1] + 1 and len(rec.got) == 2 and (rec.got[1] == eos).all()


@pytest.mark.parametrize("left", [False, True])
@pytest.mark.parametrize("kw", [dict(repetition_penalty=1.8), dict(repetition_penalty=0.5, frequency_penalty=0.3)])
def test_padding_is_no_part_of_the_prompt(case, left, kw):
    """What a row is padded with is not penalised: the scores are the raw logits of the same padded batch with the penalties of the tokens that the mask leaves.  Padded behind
    its end, a row has the tokens and scores it has alone.  (Padded before its start it need not: with modal tokens the spliced mask is the text's, extended on the left.)"""
    model, ids, modal = case
    n, L = 8, ids.shape[1]
    run = lambda i, m, **more: model.generate(i, modal_inputs=m, max_new_tokens=n, ignore_eos=True, return_step_logits=True, **kw, **more)
    alone = [run(ids[b:b + 1], {"vision": modal["vision"][b:b + 1]}) for b in range(len(ids))]
    for pad in (0, int(alone[0][0][0, L]), model.config.eos_token_id):
        wide = torch.full((len(ids), L + 3), pad, dtype=ids.dtype, device=ids.device)
        mask = torch.zeros(wide.shape, dtype=torch.bool, device=ids.device)
        at = slice(3, L + 3) if left else slice(0, L)
        wide[:, at], mask[:, at] = ids, True
        res, lg = run(wide, modal, attention_mask=mask)
        new = res[:, L + 3:]
        _, raw = model.generate(wide, modal_inputs=modal, attention_mask=mask, max_new_tokens=n, ignore_eos=True, forced_ids=new, return_step_logits=True)
        want = _processed(raw.cpu(), ids.cpu(), new.cpu(), kw["repetition_penalty"], 0.0, kw.get("frequency_penalty", 0.0), {})
        # four fp32 roundings at most, as in test_chosen_tokens_and_scores
        mag = raw.cpu().double().abs() * 2 + want.abs() + 3 * n * kw.get("frequency_penalty", 0.0)
        assert ((lg.cpu().double() - want).abs() <= 4 * 2.0 ** -24 * mag).all(), pad
        if not left:
            for b, (r, l) in enumerate(alone):
                assert torch.equal(new[b], r[0, L:]) and torch.equal(lg[b], l[0])
