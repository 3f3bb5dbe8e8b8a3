"""Worker of the tensor-parallel test of a 4-bit cache (CPU, gloo): every rank asks the cut replica for several answers of each
prompt, and the first one also asks a scheduler of its own that is not cut.  Launched by torchrun."""

import argparse
import json
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))))

import torch  # noqa: E402


class Tok:
    stop_ids = [1]

    def decode(self, ids, skip_special_tokens=True):
        return "".join(f"<{i}>" for i in ids)


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--out", required=True)
    args = ap.parse_args()

    from astrai_b200.config import AutoRegressiveLMConfig
    from astrai_b200.inference import InferenceScheduler
    from astrai_b200.models import AutoRegressiveLM
    from astrai_b200.parallel.setup import setup_parallel

    rank, world, local = int(os.environ["RANK"]), int(os.environ["WORLD_SIZE"]), int(os.environ["LOCAL_RANK"])
    cfg = AutoRegressiveLMConfig(vocab_size=512, hidden_size=128, num_hidden_layers=2, rms_norm_eps=1e-6, intermediate_size=128,
                                 tie_word_embeddings=True, max_position_embeddings=256, rope_theta=10000.0,
                                 num_attention_heads=4, num_key_value_heads=2)
    prompts = [[10 + 3 * i + j for j in range(4 + 5 * i)] for i in range(4)]
    kw = dict(max_batch_size=16, max_seq_len=128, enable_cuda_graph=False, page_size=4, kv_dtype="int4")

    def build():
        torch.manual_seed(5)
        return AutoRegressiveLM(cfg).eval()

    with setup_parallel(rank, world, local, "gloo", os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"], "cpu"):
        res = {}
        if rank == 0:
            res["alone"] = InferenceScheduler(build(), Tok(), **kw).run_batch(prompts, max_tokens=8, temperature=0.0, samples_per_prompt=3)
        sched = InferenceScheduler(build(), Tok(), tp_size=world, **kw)
        st = sched.cache.storage
        res["pool"] = [list(t.shape[2:]) for t in st.pools()]
        res["greedy"] = sched.run_batch(prompts, max_tokens=8, temperature=0.0, samples_per_prompt=3)
        torch.manual_seed(100 + rank)  # the ranks' random streams differ: the first one's decides
        res["sampled"] = sched.run_batch(prompts, max_tokens=8, temperature=1.0, top_k=40, samples_per_prompt=3)
        res["chunked"] = InferenceScheduler(sched._executor.model, Tok(), tp_size=world, chunked_prefill=True, max_prefill_tokens=5,
                                            **kw).run_batch(prompts, max_tokens=8, temperature=0.0, samples_per_prompt=2)
        with open(f"{args.out}.{rank}", "w") as fh:
            json.dump(res, fh)


if __name__ == "__main__":
    main()
