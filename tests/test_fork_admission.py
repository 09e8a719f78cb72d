"""Completions of one prompt are admitted as every request is: by the policy, above the watermark, as forks where the prompt is in the
cache."""
import pytest

from iitj_llm_coopt_b200.engine import StaticPolicy
from test_fork import engine, run

PROMPT = [(5 * i + 11) % 320 for i in range(33)]


def with_policy(eng, policy):
    eng.policy = eng.scheduler.policy = policy
    return eng


class AtMost(StaticPolicy):
    """Lets a request in only while fewer than `most` run."""
    most, asked = 2, 0

    def admit(self, seq, engine):
        self.asked += 1
        return len(engine.scheduler.running) <= self.most - 1


@pytest.mark.parametrize("lookahead", [False, True])
def test_a_policy_that_refuses_is_heard_for_every_completion(lookahead):
    want = run(engine(num_pages=96), [(5, PROMPT, 6, 0.8, 70)])
    eng = with_policy(engine(num_pages=96, lookahead=lookahead), AtMost(max_num_seqs=6, max_batched_tokens=64))
    seqs = eng.new_sequences(5, PROMPT, 6, 0.8, True, 70)
    most = 0
    while eng.has_work():
        eng.step()
        eng.cache.check()
        most = max(most, len(eng.scheduler.running))
    assert most == 2 and eng.policy.asked >= 5
    assert [[s.tokens[33:] for s in seqs]] == want


def test_the_watermark_holds_for_forks():
    # the prompt takes 5 pages of 12, a completion 1 more; 3 are kept free: 4 of the 7 fit beside the first, the rest wait
    eng = with_policy(engine(num_pages=12, max_num_seqs=9), StaticPolicy(max_num_seqs=9, max_batched_tokens=64, watermark=0.25))
    seqs = eng.new_sequences(8, PROMPT, 6, 0.8, True, 70)
    least, most = 12, 0
    while eng.has_work():
        eng.step()
        eng.cache.check()
        least, most = min(least, eng.cache.num_free), max(most, len(eng.scheduler.running))
    assert least == 3 and most == 5 and eng.counters["num_preemptions_total"] == 0
    assert [s.tokens[33:] for s in seqs] == run(engine(num_pages=96, max_num_seqs=9), [(8, PROMPT, 6, 0.8, 70)])[0]


def test_a_policy_picks_among_completions_too():
    class Last(StaticPolicy):
        def pick_next(self, waiting, engine):
            return len(waiting) - 1
    eng = with_policy(engine(num_pages=96), Last(max_num_seqs=6, max_batched_tokens=64))
    first = eng.new_sequences(3, PROMPT, 6, 0.8, True, 70)
    eng.step()
    other = eng.new_sequence(PROMPT[:9], 4, ignore_eos=True)
    eng.step()
    assert eng.scheduler.running == [first[0], other, first[2], first[1]]
    eng.run_until_done()
