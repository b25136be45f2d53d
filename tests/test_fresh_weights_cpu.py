"""Products read weights before the kernel in front has ended: the first one behind a writer of weights is an ordinary launch, on the writer's stream, whichever
thread makes it and whatever was launched in between (csrc/fresh_weights.h)."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.join(os.path.dirname(__file__), "..")
CSRC = os.path.join(ROOT, "kubernetes-gpu-cluster_b200", "csrc")


def source(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_streams_threads_and_recordings(tmp_path):
    exe = str(tmp_path / "fresh")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I", CSRC, os.path.join(ROOT, "tests", "cpp", "fresh_weights.cc"), "-o", exe,
                    "-lpthread"], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and "checks" in out.stdout, out.stdout + out.stderr


def test_the_writer_says_so_and_products_ask():
    """The writer of weights names its stream behind its launch; the products that read weights early ask for theirs, and no flag of a thread stands for it."""
    quant = source("fp8_quant.cu")
    body = quant[quant.index("KGE_API(kge_fp8_quant_weight)"):]
    assert body.index("launch_pdl(fp8_quant_weight_kernel") < body.index("pdl_weights_written((cudaStream_t)stream)") and "pdl_break_next" not in quant
    gemm = source("gemm_fp8.cu")
    stream = gemm[gemm.index("static int launch_stream("):gemm.index("static int launch_pairs(")]
    assert "p.offsets ? pdl_for_this_launch() : pdl_for_weights(st)" in stream
    # the others wait for the kernel in front before they read anything
    pair = gemm[gemm.index("fp8_pair_kernel(const __grid"):gemm.index("static int encode_map(")]
    assert pair.index("\n  pdl_wait();") < pair.index("load_box2(") and pair.index("\n  pdl_wait();") < pair.index(".ask(")
