"""Launch shapes of the attention over prompts (csrc/prompt_plan.h), on the host."""
import os
import subprocess

from test_gpu_prompt_wide import COUNTS, DIMS, GROUP, HEADS

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda-kmeans_amd", "csrc")


def run(tmp_path, body):
    """What a program of that body, with prompt_plan.h before it, prints."""
    source, program = tmp_path / "plan.cpp", tmp_path / "plan"
    source.write_text('#include "prompt_plan.h"\n#include <cstdio>\n#include <initializer_list>\nusing namespace kmx;\nint main()\n{\n%s\n}\n' % body)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", CSRC, str(source), "-o", str(program)], check=True)
    return subprocess.run([str(program)], capture_output=True, text=True, check=True).stdout


def test_batches_with_many_rows_are_taken_by_eight_wavefronts(tmp_path):
    """The batches of tests/test_gpu_prompt_wide.py, whose bound on queries is all rows, on the 256 compute units of the card; one sequence of them alone is not."""
    queries = sum(COUNTS) + 1
    shape = "plan_prompt(PromptShape{ %d / 32, %d, %d, %d, %d, 333, 256 }).wide"
    for dim in DIMS:
        got = run(tmp_path, 'printf("%%d %%d", %s, %s);' % (shape % (dim, HEADS, GROUP, len(COUNTS), queries), shape % (dim, HEADS, GROUP, 1, 300)))
        assert got == "1 0", dim


def test_no_launch_has_more_threads_than_a_launch_may(tmp_path):
    """Fewer than 2^32 threads, also where a loose bound on queries asks for a work-group of each 128 (or 256) rows of every sequence."""
    got = run(tmp_path, """
	for (uint32_t J = 1; J <= 8; ++J)
		for (uint32_t heads : { 1u, 8u, 64u })
			for (uint32_t sequences : { 1u, 255u, 256u, 512u, 1023u, 1024u, 65536u })
				for (uint32_t queries : { 1u, 31u, 8192u, 1u << 20, (1u << 20) + 1, 1u << 23, 0x7FFFFF00u }) {
					const PromptPlan p = plan_prompt(PromptShape{ J, heads, 4, sequences, queries, 5000, 256 });
					const double threads = (double)p.units * p.parts * (p.wide ? 512 : 256);
					if (prompt_launches(p) != (p.units && threads < 4294967296.0)) return printf("%u %u %u %u", J, heads, sequences, queries), 0;
					const double rows = 4.0 * queries * heads * sequences;
					if (rows < 2147483648.0 - 256.0 * heads * sequences && !prompt_launches(p)) return printf("refused %u %u %u %u", J, heads, sequences, queries), 0;
				}
	printf("fine %d", (int)prompt_launches(plan_prompt(PromptShape{ 2, 1, 4, 512, 1u << 20, 5000, 256 })));""")
    assert got == "fine 0"
