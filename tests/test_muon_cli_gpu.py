"""distill.py with the student's projections under Muon and the teacher's in 8-bit integers: trained by replayed graphs,
saved, resumed."""
import copy
import json
import math
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]


def _run(args):
    r = subprocess.run([sys.executable] + [str(a) for a in args], cwd=str(ROOT), capture_output=True, text=True, timeout=110,
                       env=dict(os.environ, HSA_ENABLE_IPC_MODE_LEGACY="0"))
    assert r.returncode == 0, (args, r.stdout[-2000:], r.stderr[-4000:])


def test_distill_with_muon_and_an_int8_teacher(tmp_path):
    from dphubert_amd.synthetic import HUBERT_BASE_CONFIG
    from dphubert_amd.trainer import seeded_model
    cfg = copy.deepcopy(HUBERT_BASE_CONFIG)
    cfg.update(encoder_num_layers=2, encoder_use_attention=[True] * 2, encoder_use_feed_forward=[True] * 2,
               encoder_num_heads=[12] * 2, encoder_ff_interm_features=[1024] * 2)
    teacher = tmp_path / "teacher.pth"
    torch.save({"config": cfg, "state_dict": seeded_model(cfg, 0).state_dict()}, teacher)
    exp = tmp_path / "exp"
    args = ["distill.py", "--gpus", "1", "--warmup_updates", "1", "--distill_layers", "0.1,2", "--log_interval", "1",
            "--teacher_ckpt", teacher, "--student_ckpt", teacher, "--exp_dir", exp, "--sparsity_warmup_updates", "2",
            "--target_sparsity", "0.5", "--synthetic_utterances", "4", "--synthetic_seconds", "2", "--optimizer", "muon",
            "--muon_momentum", "0.9", "--teacher_int8"]
    _run(args + ["--max_updates", "6"])
    ck = exp / "ckpts" / "last.ckpt"
    state = torch.load(ck, map_location="cpu", weights_only=True)
    assert state["global_step"] == 6
    opt = state["optimizer"]
    group = [g for g in opt["param_groups"] if g.get("muon")]
    assert len(group) == 1 and group[0]["momentum"] == 0.9 and len(group[0]["params"]) == 12
    assert all(set(opt["state"][i]) == {"momentum_buffer", "step"} and opt["state"][i]["momentum_buffer"].any()
               for i in group[0]["params"])
    first = torch.load(teacher, weights_only=True)["state_dict"]
    name = "encoder.transformer.layers.0.attention.q_proj.weight"
    now = {k: v for k, v in state["state_dict"].items() if k.endswith("student_model." + name)}
    assert len(now) == 1 and all(v.isfinite().all() and not torch.equal(v, first[name]) for v in now.values())
    _run(args + ["--max_updates", "8", "--resume_checkpoint", ck])
    assert torch.load(ck, map_location="cpu", weights_only=True)["global_step"] == 8
    recs = [json.loads(x) for x in (exp / "log.jsonl").read_text().splitlines() if x.strip()]
    losses = [r["train_loss"] for r in recs if "train_loss" in r]
    # (of either sign: the pruning constraint's Lagrange term is in it)
    assert losses and all(math.isfinite(v) for v in losses)
