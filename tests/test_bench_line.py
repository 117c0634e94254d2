"""`bench.py`'s line and side file with the reference chains that are in the checkout (test_gpu_chain.py states the contract for the whole
set of eleven and is skipped where two of them are absent)."""
import os

import pytest

from conftest import GOLDEN, chains_absent
from synth import CHAIN_CHIKUSEI, CHAIN_LONG_SET, CHAIN_SET
from test_gpu_chain import _run_bench

KEYS = ("metric", "value", "unit", "n_gpus", "steps", "warmup", "ms_per_step", "higher_is_better", "scaling", "vs_baseline", "dtype", "data", "config",
        "roofline", "cpu_baseline", "parity")


def expected():
    """Names of the chains that the headline mode walks: every fixture of the set whose file is here."""
    names = [(c, "chain.npz" if c == ("synth", 0, 20) else os.path.join("chains", "%s_n%d_T%d.npz" % c)) for c in CHAIN_SET + CHAIN_LONG_SET]
    names.append((("chi",) + CHAIN_CHIKUSEI, os.path.join("chains", "chi_%s_n%d_T%d.npz" % CHAIN_CHIKUSEI)))
    return [c for c, f in names if os.path.exists(os.path.join(GOLDEN, f))]


def test_only_the_two_known_chains_may_be_absent():
    assert len(expected()) == 11 - len(chains_absent()) >= 9


@pytest.mark.gpu
def test_bench_line_over_the_chains_that_are_here(tmp_path):
    last, d, side = _run_bench(tmp_path, "--patches", "12", "--steps", "20", "--warmup", "5")
    assert len(last.encode()) <= 4096 and not [k for k in KEYS if k not in d]
    assert (d["steps"], d["warmup"], d["n_gpus"], d["scaling"], d["dtype"]) == (20, 5, 1, "weak", "fp16")
    cfg = d["config"]
    assert cfg["batch_per_gpu"] == 60 and abs(d["value"] - 20 * 60 / (d["ms_per_step"] * 20e-3)) < 1e-3 * d["value"]
    # the chain's wide steps are in `value` and `ms_per_step` (the per-chain mix), not in the window that was timed
    assert cfg["wide_set_steps_in_window"] == 0 and cfg["value_is"].startswith("per-chain mix") and cfg["steps_per_chain_wide_sets"] == {"fp32": 1, "fp32h": 7}
    assert d["value"] == cfg["value_chain_mix"] < cfg["value_window"] and d["ms_per_step"] == cfg["ms_per_step_chain_mix"] > cfg["ms_per_step_window"]
    rf = d["roofline"]
    assert rf["bound"] == "mfma" and 0.05 < rf["frac"] < 1.0 and abs(rf["frac"] - rf["achieved"] / rf["peak"]) < 1e-3
    assert rf["launches"] >= 1 and rf["conv_v3_family"]["launches"] == 10 and rf["fused_resnetblock_hbm_frac"] < rf["resnetblock_launch_hbm_frac"]
    par = d["parity"]
    assert par["mode"] == "fp16" and par["n_fixtures"] == len(expected()) == len(side["parity"]["fp16"]["fixtures"])
    assert par["meets_north_star_with_sam_on_common_support"] is True
    assert par["meets_north_star"] is (par["dSAM_deg"] <= 1e-3) and par["meets_north_star"] is (par["strict_sam_misses"] == []) is d["meets_north_star"]
    assert par["latents_rel_err"] <= par["latents_rel_err_unsaturated"] < 1e-3 and par["cube_rel_err"] < 1e-3 and par["dPSNR_dB"] <= 0.01
    assert par["dSAM_unclamped_deg"] <= 1e-3 and par["dSAM_deg_on_common_support"] <= 1e-3 and any("T1000" in k for k in par["worst_of"])
    cb = d["cpu_baseline"]
    assert cb["kind"] == "port" and cb["cores"] >= 1 and 0 < cb["value"] == cb["cases"]["batch_1"]["value"] < d["value"]
    assert side["line"] == d and len(side["roofline"]["kernels"]) >= 8 and side["bf16_mode"] is None
