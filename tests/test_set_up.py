"""What launchers set up once on each device, when several threads call them for the first time at once."""
import os
import subprocess
import sys
import textwrap

import pytest

from fastgguf_b200.csrc import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include "set_up.h"
#include <chrono>
#include <cstdio>
#include <thread>
#include <vector>

static FgPerDevice state;
static std::atomic<int> began[2], ended[2], early, failed;

int main() {
    // sixteen threads at a time on two devices: one set-up each, and nobody goes on before it has ended
    std::vector<std::thread> threads;
    for (int i = 0; i < 16; i++)
        threads.emplace_back([i] {
            const int dev = i % 2;
            const int code = fg_set_up_on(state, dev, [dev] {
                began[dev]++;
                std::this_thread::sleep_for(std::chrono::milliseconds(50));
                ended[dev]++;
                return 0;
            });
            if (code) failed++;
            if (ended[dev] != 1) early++;
        });
    for (auto &t : threads) t.join();
    if (began[0] != 1 || began[1] != 1 || early || failed) return printf("%d %d set-ups, %d early, %d failed\n", (int)began[0], (int)began[1], (int)early, (int)failed), 1;
    // a set-up that fails says so each time, until one succeeds
    int tries = 0;
    auto third = [&] { return ++tries < 3 ? 7 : 0; };
    for (int want : {7, 7, 0, 0})
        if (fg_set_up_on(state, 5, third) != want) return printf("try %d\n", tries), 1;
    if (tries != 3) return printf("%d tries\n", tries), 1;
    // devices past the table are set up in every call
    for (int i = 0; i < 2; i++) fg_set_up_on(state, 64, third);
    return tries == 5 ? 0 : (printf("%d tries past the table\n", tries), 1);
}
"""


def test_one_thread_sets_up_and_the_others_wait(tmp_path):
    src, exe = tmp_path / "set_up.cpp", tmp_path / "set_up"
    src.write_text(PROGRAM)
    p = subprocess.run(["g++", "-O1", "-std=c++17", "-pthread", "-I", build.CSRC_DIR, str(src), "-o", str(exe)], capture_output=True, text=True)
    assert p.returncode == 0, p.stderr
    p = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert p.returncode == 0, p.stdout


FIRST_CALLS = """
    import sys, threading
    import torch
    from fastgguf_b200 import ops
    from fastgguf_b200.ops import fast_gemm
    g = torch.Generator(device="cuda").manual_seed(1)
    def random(*shape):
        return torch.randn(*shape, generator=g, device="cuda") * shape[-1] ** -0.5
    CALLS
    calls = [(k, i) for i in range(4) for k in kinds] * 2
    together, got, wrong = threading.Barrier(len(calls)), [None] * len(calls), []

    def run(j):
        k, i = calls[j]
        with torch.cuda.stream(torch.cuda.Stream()):
            together.wait()
            try:
                got[j] = k(i)
            except Exception as e:
                wrong.append(repr(e))
            torch.cuda.current_stream().synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=run, args=(j,)) for j in range(len(calls))]
    for t in threads: t.start()
    for t in threads: t.join()
    ops.raise_on_device_error("first calls")
    if not wrong:
        wrong = [f"call {j} differs" for j, (k, i) in enumerate(calls) if not torch.equal(got[j], k(i))]
    sys.exit("; ".join(wrong) if wrong else 0)
"""
KINDS = {
    "mxfp4": """
    w, stack = ops.mxfp4_quantize(random(1000, 2048)), ops.mxfp4_quantize(random(2, 1000, 2048))
    xs = [random(m, 2048).bfloat16() for m in (1, 12, 70, 300)]
    packed = [ops.mxfp4_quantize(x) for x in xs]
    cuts = [torch.tensor([0, x.shape[0] // 2, x.shape[0]], dtype=torch.int32, device="cuda") for x in xs]
    kinds = [lambda i: ops.gemm_mxfp4(xs[i], w), lambda i: ops.gemm_mxfp4_both(packed[i], w), lambda i: ops.gemm_mxfp4_grouped(xs[i], stack, cuts[i])]
""",
    "gemm": """
    w, wide = random(1024, 2048).bfloat16(), random(1024, 2048)
    xs, x32 = [random(m, 2048).bfloat16() for m in (1, 40, 300, 1500)], [random(m, 2048) for m in (1, 16, 40, 300)]
    kinds = [lambda i: fast_gemm.gemm_tc(xs[i], w), lambda i: fast_gemm.gemm_tc(xs[i], w, out_dtype=torch.float32),
             lambda i: fast_gemm.gemm_f32_stream(x32[i], wide) if i < 2 else fast_gemm.gemm_f32(x32[i], wide)]
""",
}


@pytest.mark.gpu
@pytest.mark.parametrize("which", list(KINDS))
@pytest.mark.parametrize("attempt", range(3))
def test_first_calls_of_many_threads_at_once(which, attempt):
    program = textwrap.dedent(FIRST_CALLS.replace("    CALLS\n", KINDS[which].lstrip("\n")))
    p = subprocess.run([sys.executable, "-c", program], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert p.returncode == 0, p.stderr[-2000:]
