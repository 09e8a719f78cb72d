"""How often the prompt of several completions is computed when there is not room for all of them at once."""
import pytest

from test_fork import engine, run

PROMPT = [(5 * i + 11) % 320 for i in range(30)]


def counted(eng, groups):
    out = run(eng, groups)
    return out, eng.counters["prompt_tokens_total"]


@pytest.mark.parametrize("kw", [dict(max_num_seqs=4), dict(max_num_seqs=2), dict(max_num_seqs=4, max_num_batched_tokens=7)])
def test_more_completions_than_slots_compute_the_prompt_once(kw):
    groups = [(8, PROMPT, 6, 0.8, 70)]
    want = run(engine(num_pages=96, max_num_seqs=9), groups)
    assert counted(engine(num_pages=96, **kw), groups) == (want, 30)


def test_prompts_do_not_take_the_slots_of_each_others_completions():
    groups = [(4, [(t + 7 * j) % 320 for t in PROMPT], 6, 0.8, 70 + j) for j in range(4)]
    want = run(engine(num_pages=96, max_num_seqs=16, max_num_batched_tokens=256), groups)
    for slots in (4, 6):
        got, computed = counted(engine(num_pages=96, max_num_seqs=slots), groups)
        # (a prompt's last portion of one token is a decode, which this counter does not count: up to one for each prompt)
        assert got == want and 116 <= computed <= 120


def test_a_preempted_completion_shares_again():
    groups = [(3, PROMPT[:25], 30, 0.8, 70)]
    want = run(engine(num_pages=96), groups)
    eng = engine(num_pages=12)                         # 3 pages of prompt, 4 more each: not enough for all three
    got, computed = counted(eng, groups)
    assert got == want and eng.counters["num_preemptions_total"] > 0
    # (what the preempted one had generated is fed again, the prompt is not)
    assert computed <= 25 + eng.counters["num_preemptions_total"] * 30


def test_requests_behind_a_prompt_of_many_completions_are_not_kept_out_for_good():
    eng = engine(num_pages=96, max_num_seqs=3)
    many = eng.new_sequences(7, PROMPT, 6, 0.8, True, 70)
    other = eng.new_sequence(PROMPT[:9], 4, ignore_eos=True)
    eng.run_until_done()
    assert other.finished and all(s.finished for s in many) and eng.counters["prompt_tokens_total"] == 39
