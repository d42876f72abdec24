import sys, time
import os; sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import torch
from adt_str_amd.network import ADTModel, ADTModelConfig
torch.manual_seed(0)
m = ADTModel(ADTModelConfig(input_sec=10.0, time_res=0.01, win_length=2048, sample_rate=16000, enc_layers=4, dec_layers=4, nhead=6, d_query=128,
                            dropout=0.1, tgt_vocab_size=1400, plain=True, n_mels=128)).cuda().eval()
# python tools/bench_decode.py [clips] [precision] [kv_bits]
B0, precision, kv_bits = int(sys.argv[1]) if len(sys.argv) > 1 else 8, sys.argv[2] if len(sys.argv) > 2 else "bf16", int(sys.argv[3]) if len(sys.argv) > 3 else 16
m.set_precision(precision)
src = torch.randn(B0, 160000, device="cuda") * 0.1
eng = m.engine
for mode in ("graph", "cached", "full") if kv_bits == 16 else ("graph", "cached"):
    for L in (64, 256, 1000):
        if mode == "full" and L > 256:
            continue
        m.sample(src, None, None, max_length=8, use_cache=mode != "full")
        torch.cuda.synchronize(); t0 = time.perf_counter()
        if mode == "full":
            out = m.sample(src, None, None, max_length=L, end_token=-1, use_cache=False)     # end_token -1: never finishes -> L-1 steps
        else:
            mem16, B, S = eng.encode(src)
            out = eng.greedy_decode_cached(mem16, B, S, L, 2, -1, use_graph=mode == "graph", kv_bits=kv_bits)
        torch.cuda.synchronize(); dt = time.perf_counter() - t0
        print(f"{mode:7s} max_length={L}: {dt*1e3:.1f} ms  ({dt/(L-1)*1e3:.3f} ms/step), out {tuple(out.shape)}")
