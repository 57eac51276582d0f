"""One rank of the tensor-parallel test of tree decoding (started by test_tree_tp_gpu.py, one process per rank; the ranks share the visible GPUs).
Prints the tokens of the small end-to-end fixture case, decoded in drafted trees after the prefill."""
import json
import os
import random
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path[:0] = [HERE, os.path.dirname(HERE)]
import torch
import torch.distributed as dist


def main():
    import faulthandler

    faulthandler.dump_traceback_later(100, exit=True)  # a stuck rank says where, then leaves
    rank, world = int(os.environ["RANK"]), int(os.environ["WORLD_SIZE"])
    torch.set_num_threads(2)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    dev = torch.device("cuda", rank % torch.cuda.device_count())
    torch.cuda.set_device(dev)

    import golden_cases as gc
    from oracle import gen_golden as gg
    from mini_sglang_amd import comm
    from mini_sglang_amd.mem_cache import MHAKVPool, PageAllocator, ReqToTokenPool
    from mini_sglang_amd.runtime.batch_info import BatchInfo, Req, SamplingParams
    from mini_sglang_amd.runtime.model_runner import ModelConfig, ModelRunner, ServerArgs
    from mini_sglang_amd.runtime.qwen3 import Qwen3Config
    from mini_sglang_amd.runtime.tree_decode import TreeDecoder

    cfg_kw, ps, (pseed, plens), _, wseed, wstd, estd, succ = gg.E2E_CASES["tiny_ps16"]
    cfg = Qwen3Config(**cfg_kw)
    args = ServerArgs(page_size=ps, device=str(dev), disable_cuda_graph=True, max_num_reqs=8, random_seed=wseed, weight_std=wstd, embed_std=estd,
                      successor_head=succ)
    pages = 1024 // ps
    r2t = ReqToTokenPool(8, cfg.max_position_embeddings, ps, str(dev))
    pa = PageAllocator(pages, ps)
    kv = MHAKVPool(pages * ps, ps, torch.bfloat16, cfg.num_key_value_heads // world, cfg.head_dim, cfg.num_hidden_layers, str(dev))
    mr = ModelRunner(ModelConfig(cfg), args, gpu_id=dev.index, tp_rank=rank, tp_size=world, req_to_token_pool=r2t, page_allocator=pa, kv_cache_pool=kv)
    ar = comm.enable_xgmi_allreduce(max_bytes=1 << 20)
    prompts = gg.e2e_prompts(pseed, plens, cfg.vocab_size)
    reqs = [Req(i, p, SamplingParams(0.0)) for i, p in enumerate(prompts)]
    batch = BatchInfo.init_new(reqs, r2t, pa, kv)
    batch.prepare_for_extend()
    logits, _ = mr.forward_generate(batch)
    mr.process_result(batch, logits)
    ar.check()
    dec = TreeDecoder(mr, batch, 5, max_new_tokens=64, logprobs=3, use_graph=False)   # (the ranks' exchange over the host cannot be captured)
    rng, truth, steps = random.Random(7), gc.load("e2e_tiny_ps16.pt")["tokens"][:, :24].tolist(), 0
    while min(len(r.token_ids) - len(p) for r, p in zip(reqs, prompts)) < 24:
        drafts = []
        for r, p, t in zip(reqs, prompts, truth):
            done = len(r.token_ids) - len(p)
            right = t[done: done + rng.randint(0, 3)]
            drafts.append((right + [rng.randrange(cfg.vocab_size) for _ in range(4 - len(right))], [0, 1, 2, 0]))
        got = dec.step(drafts)
        for new, scores in zip(got, dec.last_logprobs):
            assert [ids[0] for _, _, ids, _ in scores] == new   # the most probable token is the greedy one
        ar.check()
        steps += 1
    dec.sync_host()
    print("STEPS %d" % steps)
    print("TOKENS " + json.dumps([r.token_ids[len(p): len(p) + 24] for r, p in zip(reqs, prompts)]), flush=True)
    comm.disable_xgmi_allreduce()
    dist.destroy_process_group()


if __name__ == "__main__":
    main()
