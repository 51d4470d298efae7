"""The command's several texts beside a training."""
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu


def train(bmb, tmp_path, *more):
    text = tmp_path / "t.txt"
    text.write_text("the quick brown fox jumps over the lazy dog\n" * 60)
    exe = os.path.join(os.path.dirname(bmb.LIB_PATH), "bmb_train_gpt")
    return subprocess.run([exe, "-d", str(text), "-n", "2", "-b", "1", "-t", "32", "-l", "1", "--eval", "0", "--eval-batches", "1", "--sample", "0", "--save", "", *more],
                          capture_output=True, text=True, timeout=120)


@pytest.mark.parametrize("bad,why", [(("--heads", "1", "--embd", "96", "--texts", "2"), "head size 96"), (("--heads", "2", "--embd", "64", "--repetition", "0"), "bad argument"),
                                     (("--heads", "2", "--embd", "64", "--texts", "2", "--temp", "0"), "bad argument")])
def test_what_drawing_refuses_is_told_before_the_training(bmb, cuda, tmp_path, bad, why):
    got = train(bmb, tmp_path, "--unfused", "--len", "20", *bad)
    assert got.returncode == 1 and why in got.stderr and "step " not in got.stdout, got


def test_several_texts_behind_a_training(bmb, cuda, tmp_path):
    got = train(bmb, tmp_path, "--heads", "2", "--embd", "64", "--texts", "3", "--presence", "0.3", "--len", "400")
    assert got.returncode == 0 and "final  train loss" in got.stdout and "[text 3]" in got.stdout, got
    got = train(bmb, tmp_path, "--heads", "1", "--embd", "96", "--unfused", "--len", "20")           # (one text goes another way, with any head size)
    assert got.returncode == 0 and "final sample" in got.stdout, got
