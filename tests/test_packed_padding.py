"""Decode steps that are padded to a size of the captured graphs' ladder, over a packed cache."""
import torch

import kv4_plain as P
from configs import TINY_B
from iitj_llm_coopt_b200 import EngineConfig, LlamaConfig, build_engine
from iitj_llm_coopt_b200.engine import StepEntry


class Watched(P.PackedTorchKernels):
    """Notes the slots that are stored to."""

    def __init__(self):
        super().__init__()
        self.slots = []

    def rope_store_kv4(self, qkv, tables, slots, *args, **kw):
        self.slots.append(slots.clone())
        return super().rope_store_kv4(qkv, tables, slots, *args, **kw)


def test_padding_rows_store_nothing():
    rows = {}
    for padded in (False, True):
        kernels = Watched()
        eng = build_engine(None, EngineConfig(dtype="float32", page_size=8, num_pages=32, device="cpu", max_num_seqs=9,
                                              max_num_batched_tokens=128, kv_cache="int4"),
                           config=LlamaConfig.from_dict(TINY_B), random_seed=3, kernels=kernels)
        for r in range(9):
            eng.cache.admit(r)
        eng.runner.step([StepEntry(r, [(7 * i + r) % 300 for i in range(5 + r)], []) for r in range(9)])
        kernels.slots.clear()
        eng.runner.use_graphs = padded                 # (nothing is captured before a shape has come up three times)
        rows[padded] = eng.runner.step([StepEntry(r, [11 + r], [0]) for r in range(9)])
        assert eng.runner.padded_steps == int(padded) and len(kernels.slots) == len(eng.runner.model.layers)
        for slots in kernels.slots:
            kept = slots[slots >= 0]
            assert len(slots) == (16 if padded else 9) and len(kept) == 9 and len(set(kept.tolist())) == 9      # each slot once
        for g in eng.cache.paged:
            assert not eng.cache.groups[g].storage[:, -1].any()        # the padding page
    # (products of 9 and of 16 rows add in another order, 2^-24 of a few hundred numbers at a time; a code beside it where one lies that
    # near a border moves one number of thousands by a fifteenth of its group's spread)
    assert ((rows[False] - rows[True]).norm(dim=-1) / rows[False].norm(dim=-1)).max() < 5e-3
