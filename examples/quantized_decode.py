"""A prompt compressed by the CORE step, its kept rows in 4 bits, and decoding over them.

One layer of Llama-3.1-8B's shape on seeded synthetic inputs: the compression step
scores a 16384-token prompt and keeps a quarter of it; the kept rows are picked and
quantised in one pass; each decoded token is quantised behind them, attended to
as codes, and gets the latent memory's readout added.  Printed: bytes of the kept
cache, the error against the same steps over the unquantised rows, time per token.

    python examples/quantized_decode.py [--bits 4|8] [--group 32|64|128]
"""

import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

from core_b200 import engine, ops, synthetic  # noqa: E402
from core_b200.kvcache import QuantizedKV  # noqa: E402

HQ, HKV, D, L, NQ, D_MEM, STEPS = 32, 8, 128, 16384, 128, 512, 64


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--bits", type=int, default=4, choices=(4, 8))
    ap.add_argument("--group", type=int, default=64, choices=(32, 64, 128))
    a = ap.parse_args()
    dev = torch.device("cuda", 0)
    q, k, v = synthetic.make_layer_inputs(seed=0, batch=1, n_kv_heads=HKV, n_q_heads=HQ, seq_len=L,
                                          n_queries=NQ, device=dev)
    w = synthetic.make_layer_weights(seed=1, n_kv_heads=HKV, n_q_heads=HQ, d_mem=D_MEM, hidden=HQ * D)
    lw = engine.LayerWeights.prepare(geometry=w["geometry"], prototypes=w["prototypes"], hadamard=w["hadamard"],
                                     mlp_params=w["mlp"], theta=w["theta"], gate=w["gate"], n_kv_heads=HKV,
                                     n_q_heads=HQ, device=dev)
    memory = engine.MemoryState.zeros(1, D_MEM, HKV * D, dev)
    n_kept = engine.n_kept_for(L, 0.75, 4)
    step = engine.compress_layer(q, k, v, lw, n_kept=n_kept, positions=torch.arange(L, device=dev)[None],
                                 original_length=L, is_prefill=True, memory=memory)

    cache = QuantizedKV.empty(1, HKV, n_kept + STEPS, bits=a.bits, group=a.group, device=dev)
    cache.append(k, v, index=step["keep"])  # picked and quantised in one pass
    plain_k, plain_v = step["keys"], step["values"]
    print(f"{n_kept} of {L} tokens kept: {2 * plain_k.numel() * 2 / 2**20:.1f} MiB as bf16, "
          f"{cache.nbytes / 2**20:.1f} MiB in {a.bits} bits (room for {cache.capacity})")

    o_fold = engine.fold_groups(w["o_proj"].to(dev), HKV, HQ // HKV, D)
    new = synthetic.make_layer_inputs(seed=2, batch=1, n_kv_heads=HKV, n_q_heads=HQ, seq_len=STEPS,
                                      n_queries=STEPS, device=dev)

    def decode(t):
        """One token: its row into the cache, attention over the codes, the readout."""
        qt, kt, vt = (x[:, :, t:t + 1] for x in new)
        cache.append(kt, vt)
        out, _ = cache.attend(qt)
        out = out.reshape(1, 1, HQ * D)
        return ops.memory_readout(qt, lw.theta, lw.gate, memory.M, memory.b, o_fold, out, n_kv_heads=HKV)

    worst = 0.0
    start, end = torch.cuda.Event(True), torch.cuda.Event(True)
    outs = []
    for t in range(STEPS):
        if t == 8:
            start.record()
        outs.append(decode(t))
    end.record()
    torch.cuda.synchronize()
    ops.status(dev)
    for t in range(STEPS):
        qt, kt, vt = (x[:, :, t:t + 1] for x in new)
        plain_k, plain_v = torch.cat([plain_k, kt], 2), torch.cat([plain_v, vt], 2)
        ref, _ = ops.attention_prefill(qt, plain_k, plain_v)
        ref = ops.memory_readout(qt, lw.theta, lw.gate, memory.M, memory.b, o_fold, ref.reshape(1, 1, HQ * D),
                                 n_kv_heads=HKV)
        worst = max(worst, float((outs[t].float() - ref.float()).norm() / ref.float().norm()))
    print(f"{STEPS} tokens decoded: {start.elapsed_time(end) / (STEPS - 8) * 1e3:.0f} us a token and layer; "
          f"the output differs from the unquantised rows' by {worst:.3f} of its norm at most")


if __name__ == "__main__":
    main()
