"""Steps and generations whose tokens are drawn (lg_hip_forward_sample, the sampling of the session helpers and of run-hip): against the CPU oracle's
logits and the definition in whole numbers, and with drafts against without."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from conftest import ROOT
from serving import sample_ref
from test_gpu_draft import write_head

pytestmark = pytest.mark.gpu
HOW = [(1.0, 64, 0.95, 0.0), (0.8, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.0), (1.5, 40, 1.0, 0.1), (0.0, 0, 1.0, 0.0)]


@pytest.mark.parametrize("how", HOW)
def test_drawn_steps_match_the_oracle(lg, ob, gpu_required, model_path, how):
    """The device's logits are the oracle's bit for bit, so the drawn tokens are those of the oracle's rows; drafts that are drawn again hold, the first other one
    ends the block, and the hidden state is the accepted row's."""
    path, spec = model_path("tiny_full")
    V, E, rows = spec["n_vocab"], spec["n_embd"], 5
    rng = np.random.default_rng(hash(how) % 1000)
    prompt = rng.integers(0, V, 40).astype(np.int32)
    o = ob.Oracle(path)
    gpu = lg.hiplib.HipBackend(path, 160, max_rows=rows)
    try:
        kv = o.kv_new(160, ob.I8)
        o.prefill(kv, prompt[:-1], 0, ob.I8)
        gpu.prefill(prompt[:-1], 0)
        gpu.set_option("store_logits", 1)
        tok, pos, seen = int(prompt[-1]), len(prompt) - 1, set()
        for step in range(8):
            n = 1 if step == 3 else rows
            first_bad = int(rng.integers(1, n + 1))
            us, blk, picks, hiddens = [], [tok], [], []
            for j in range(n):
                _, row, hid = o.forward(kv, blk[j], pos + j, ob.I8, want_hidden=True)
                u = np.float32(rng.random())
                while not sample_ref(row, *how, u)[3]:
                    u = np.float32(rng.random())
                us.append(u); picks.append(sample_ref(row, *how, u)[0]); hiddens.append(hid)
                if j + 1 < n:
                    blk.append(picks[j] if j + 1 < first_bad else (picks[j] + 1 + int(rng.integers(0, V - 1))) % V)
            want = 1
            while want < n and picks[want - 1] == blk[want]:
                want += 1
            print(f"drawn step {step} rows {n} pos {pos} adv {want}", flush=True)
            adv, out = gpu.forward_sample(np.array(blk, np.int32), pos, how, us)
            assert adv == want and out.tolist() == picks
            assert np.array_equal(gpu.last_hidden(E).view(np.uint32), hiddens[adv - 1].view(np.uint32))
            assert np.array_equal(gpu.logits_row(n - 1, V).view(np.uint32), row.view(np.uint32))
            seen.add(adv)
            tok, pos = picks[adv - 1], pos + adv
        assert len(seen) >= 2
        if not how[0] > 0:                                 # without a temperature it is the greedy step
            blk = np.array([tok, 1, 2], np.int32)
            assert gpu.forward_sample(blk, pos, how, [0.5] * 3)[1].tolist() == gpu.forward_spec(blk, pos)[1].tolist()
    finally:
        gpu.close(); o.close()


def test_drawn_steps_are_refused_without_logits_or_arguments(lg, gpu_required, model_path):
    path, spec = model_path("tiny")
    gpu = lg.hiplib.HipBackend(path, 64, max_rows=4)
    try:
        gpu.prefill([1, 2, 3], 0)
        with pytest.raises(lg.hiplib.HipError, match=r"store_logits.*\(code -4\)"):
            gpu.forward_sample([5], 3, HOW[0], [0.5])
        gpu.set_option("store_logits", 1)
        for toks, pos, code in (([5], 64, -2), ([5] * 5, 3, -2), ([spec["n_vocab"]], 3, -2), ([5, 5], 63, -2)):
            with pytest.raises(lg.hiplib.HipError, match=rf"\(code {code}\)"):
                gpu.forward_sample(toks, pos, HOW[0], [0.5] * len(toks))
        H, t, o, adv = gpu.H, np.array([5], np.int32), np.zeros(1, np.int32), C.c_int32(0)
        assert H.lg_hip_forward_sample(gpu.dev, gpu.dkv, t, 1, 3, None, np.zeros(1, np.float32), o, C.byref(adv)) == -1
        assert gpu.forward_sample([5], 3, HOW[0], [0.5])[0] == 1          # and the step after a refusal works
    finally:
        gpu.close()


def test_drawn_generation_is_the_same_with_and_without_drafts(lg, gpu_required, model_path, model_dir):
    """A token's number belongs to its position: blocks with perfect, wrong and absent drafts and a draft head's drafts, host-driven and in batches, give the
    tokens of one-row steps; another seed gives others, temperature 0 the greedy ones."""
    path, spec = model_path("tiny_full")
    head = write_head(lg, model_dir, "tiny_full", spec)
    rng = np.random.default_rng(6)
    prompt = rng.integers(0, spec["n_vocab"], 30).astype(np.int32)
    gpu = lg.hiplib.HipBackend(path, 160, max_rows=5)
    t = None
    try:
        def run(**how):
            gpu.new_cache(160)
            return gpu.generate(prompt, 40, **how)[0].tolist()

        greedy = run()
        t = gpu.mtp_open(head)
        gpu.sampling(1.0, 50, 0.95, 0.0, seed=11)
        plain = run()
        assert plain != greedy
        for drafts in (np.array(plain + [0] * 8), (np.array(plain + [0] * 8) + 1) % spec["n_vocab"], None):
            print("drawn generation with drafts", flush=True)
            assert run(rows=4, drafts=drafts) == plain
        gpu.new_cache(160)
        assert gpu.generate_mtp(t, prompt, 40, 4)[0].tolist() == plain
        gpu.new_cache(160)
        assert gpu.generate_mtp_rounds(t, prompt, 40, 4, 3)[0].tolist() == plain
        gpu.sampling(1.0, 50, 0.95, 0.0, seed=12)
        assert run() != plain
        gpu.sampling(1.0, 50, 0.95, 0.0, seed=11)
        assert run(rows=5, drafts=None) == plain
        gpu.sampling()
        assert run() == greedy
    finally:
        gpu.sampling()
        if t:
            gpu.mtp_close(t)
        gpu.close()


def test_run_hip_draws_and_verifies_its_own_output(lg, gpu_required, model_path, model_dir):
    path, spec = model_path("tiny_full")
    exe = os.path.join(ROOT, "little-gemma_amd", "host", "run-hip")

    def cli(*more):
        r = subprocess.run([exe, "-m", path, "-p", "1,17,23,5", "-n", "24", *more], capture_output=True, text=True, timeout=120)
        assert r.returncode == 0, r.stderr[-500:]
        return r

    how = ["-temp", "0.9", "-top-k", "40", "-top-p", "0.95", "-min-p", "0.01", "-seed", "5"]
    plain = cli(*how).stdout
    assert plain != cli().stdout and plain != cli(*how[:-1], "6").stdout
    again = cli(*how, "-mtp", "self")
    assert again.stdout == plain and "is byte-identical to plain sampled output" in again.stderr
    head = write_head(lg, model_dir, "tiny_full", spec)
    drafted = cli(*how, "-mtp", head)
    assert drafted.stdout == plain and "is byte-identical to plain sampled output" in drafted.stderr
