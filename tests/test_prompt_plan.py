"""Launch shapes of the attention over prompts (csrc/prompt_plan.h), on the host."""
import os
import subprocess

from test_gpu_prompt_wide import COUNTS, DIMS, GROUP, HEADS

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda-kmeans_amd", "csrc")


def run(tmp_path, body):
    """What a program of that body, with prompt_plan.h before it, prints."""
    source, program = tmp_path / "plan.cpp", tmp_path / "plan"
    source.write_text('#include "prompt_plan.h"\n#include <cstdio>\nusing namespace kmx;\nint main()\n{\n%s\n}\n' % body)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", CSRC, str(source), "-o", str(program)], check=True)
    return subprocess.run([str(program)], capture_output=True, text=True, check=True).stdout


def test_batches_with_many_rows_are_taken_by_eight_wavefronts(tmp_path):
    """The batches of tests/test_gpu_prompt_wide.py, whose bound on queries is all rows, on the 256 compute units of the card; one sequence of them alone is not."""
    queries = sum(COUNTS) + 1
    shape = "plan_prompt(PromptShape{ %d / 32, %d, %d, %d, %d, 333, 256 }).wide"
    for dim in DIMS:
        got = run(tmp_path, 'printf("%%d %%d", %s, %s);' % (shape % (dim, HEADS, GROUP, len(COUNTS), queries), shape % (dim, HEADS, GROUP, 1, 300)))
        assert got == "1 0", dim
