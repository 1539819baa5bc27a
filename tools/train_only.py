"""BASELINE.json config 4 and nothing else: N train.py-style steps (tests/train_replay.py: package (A) forward at 1296x840, SH1,
white background, random camera per step; fused loss epilogue; backward; densification statistics; torch Adam) at a fixed number
of Gaussians -- the command the rocprofv3 passes of tools/profile_r04.sh run.  argv: steps [P] [optimiser: torch (default), 32 or 8 =
gs_localization_amd.map_optimizer.AdamW with moments of that many bits].  Prints the time of a step and the mean losses of the steps' fifths."""
import sys, os, time
sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import torch
from tests.train_replay import TrainReplay
steps = int(sys.argv[1]) if len(sys.argv) > 1 else 40
P = int(sys.argv[2]) if len(sys.argv) > 2 else 1_500_000
tr = TrainReplay(P0=P, P1=P, densify_from=10**9)
opt = sys.argv[3] if len(sys.argv) > 3 else "torch"
if opt != "torch":
    from tests.train_replay import LRS
    from gs_localization_amd.map_optimizer import AdamW
    tr.opt = AdamW([{"params": [tr.par[k]], "lr": LRS[k], "name": k} for k in LRS], lr=0.0, eps=1e-15, state_bits=int(opt))
for it in range(1, 4):
    tr.step(it)
torch.cuda.synchronize(); t0 = time.perf_counter()
losses = [tr.step(it) for it in range(4, 4 + steps)]
torch.cuda.synchronize()
ms = 1e3 * (time.perf_counter() - t0) / steps
losses = torch.stack([x.detach().reshape(()) for x in losses]).double().cpu()
print("train steps", steps, "P", P, "optimiser", opt, "ms/step %.3f" % ms, "mean losses", " ".join("%.5f" % float(x.mean()) for x in losses.chunk(5)))
