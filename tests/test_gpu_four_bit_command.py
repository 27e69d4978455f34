"""The command line's --cache-bits: the same tokens and logits as the engine that is asked for such a cache in Python."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from tests.util import TINY, make_model_dir, random_tokens

pytestmark = pytest.mark.gpu
LEONE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bin", "leone")


def _run(*args):
    return subprocess.run([sys.executable, LEONE, *args], capture_output=True, text=True, timeout=100)


def test_generate_and_eval(tmp_path):
    from leone_amd.api import Runtime
    from leone_amd.engine.engine import Engine, StepEntry
    from leone_amd.runtime import load_model
    folder = str(tmp_path / "model")
    make_model_dir(folder, TINY["M"], seed=11, dtype=torch.bfloat16)
    vocab = TINY["M"]["vocab_size"]
    prompt = random_tokens(4, 70, vocab)
    run = _run("generate", "-m", folder, "--prompt-tokens", ",".join(map(str, prompt)), "-n", "12", "--ignore-eos", "--cache-bits", "4")
    assert run.returncode == 0, run.stderr
    runtime = Runtime.load(folder, "bfloat16", max_requests=1, cache_bits=4)
    assert [int(t) for t in run.stdout.split()] == runtime.generate_tokens([prompt], 12, eos_token_id=None)[0].tokens

    tokens_file, logits_file = tmp_path / "t.bin", tmp_path / "l.bin"
    tokens = random_tokens(5, 40, vocab)
    np.asarray(tokens, dtype="<u4").tofile(tokens_file)
    run = _run("eval", "-m", folder, "--tokens", str(tokens_file), "--window", "64", "--prefill-chunk", "39", "--logits", str(logits_file),
               "--cache-bits", "4")
    assert run.returncode == 0, run.stderr
    got = np.fromfile(logits_file, dtype="<f4").reshape(39, -1)
    model = load_model(folder, "bfloat16")
    logits = [Engine(model, max_tokens=128, max_requests=1, max_context=64, cache_bits=bits).step([StepEntry("w", tokens[:39], list(range(39)))]).logits
              for bits in (4, None)]
    small, usual = (x.float().cpu().numpy() for x in logits)
    assert np.array_equal(got, small) and not np.array_equal(got, usual)


def test_other_numbers_and_models_are_refused(tmp_path):
    folder = str(tmp_path / "model")
    make_model_dir(folder, TINY["A"], seed=1, dtype=torch.bfloat16)
    run = _run("generate", "-m", folder, "--prompt-tokens", "1,2", "-n", "2", "--cache-bits", "8")
    assert run.returncode == 2 and "--cache-bits" in run.stderr
    run = _run("generate", "-m", folder, "--prompt-tokens", "1,2", "-n", "2", "--cache-bits", "4")
    assert run.returncode != 0 and "4 bits" in run.stderr
