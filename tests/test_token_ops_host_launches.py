"""What the host code of the embedding, layer norm and token log probability entry points decides, on the CPU: as tests/test_host_launches.py,
every signed overflow an abort, launches recorded instead of made (tests/host_launches)."""
import os
import re
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from tests.test_host_launches import CHECKED, ROOT

SHAPE, WS = "-2", "-5"
THREADS = {"embedding_kernel": 256, "embedding_sum_kernel": 256, "layernorm_residual_bwd_kernel": 1024, "token_logprobs_kernel": 256,
           "token_logprobs_join_kernel": 256, "token_logprobs_bwd_kernel": 256, "layernorm_dweight_kernel": 256, "embedding_few_kernel": 1024,
           "embedding_gather_kernel": 1024, "embedding_count_kernel": 1024, "embedding_scatter_kernel": 1024, "embedding_join_kernel": 1024}


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("host")

    def compile_(name):
        obj = str(tmp / (name + ".o"))
        subprocess.check_call(["/opt/rocm/bin/hipcc", "--offload-arch=gfx950", "--offload-host-only", "-O1", "-std=c++17", "-w", *CHECKED, "-c",
                               os.path.join(ROOT, "tyr_amd", "csrc", name + ".hip"), "-o", obj])
        return obj
    with ThreadPoolExecutor() as pool:
        objs = list(pool.map(compile_, ("capi", "embedding", "layernorm", "logprobs")))
    main, exe = str(tmp / "recorder.o"), str(tmp / "recorder")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-D__HIP_PLATFORM_AMD__=1", "-isystem", "/opt/rocm/include", "-c",
                           os.path.join(ROOT, "tests", "host_launches", "token_recorder.cpp"), "-o", main])
    # what the other kernel files and the fat binaries would define is never reached
    subprocess.check_call(["/opt/rocm/llvm/bin/clang++", main, *objs, "-fsanitize=signed-integer-overflow", "-fsanitize-minimal-runtime",
                           "-Wl,--unresolved-symbols=ignore-all", "-o", exe])

    def run(lines):
        r = subprocess.run([exe], input="\n".join(lines) + "\n", capture_output=True, text=True)
        got = r.stdout.splitlines()
        assert r.returncode == 0 and len(got) == len(lines), (lines[min(len(got), len(lines) - 1)], r.returncode, r.stderr[-300:])
        return got
    return run


def launches(got):
    """[(kernel, template arguments, workgroups)]; a launch has fewer than 2^32 threads."""
    out = []
    for word in got.split()[1:]:
        m = re.fullmatch(r"(\w+)(?:<(.*)>)?:(\d+)", word)
        out.append((m[1], m[2], int(m[3])))
        assert int(m[3]) * THREADS.get(m[1], 1) < 1 << 32, got
    return out


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("d", [8, 520, 4096, 1 << 20])
def test_the_scratch_of_an_embedding_s_gradient_holds_what_its_launches_write(ask, d, bf16):
    """Pairs of 8 bytes (twice for a radix sort), a byte a token, the sort's counts, and two f32 rows a piece."""
    for n in (1, 2, 100, 2049, 32768, 32769, 200000, 1 << 22):
        for vocab in (1, 255, 262144, 262145, 1 << 20, 50000000):
            need, = ask([f"embedding_bwd_bytes {n} {vocab} {d} {bf16}"])
            calls = [f"embedding_bwd {n} {vocab} {d} {bf16} {into} {need}" for into in (0, 1)]
            for into, got in enumerate(ask(calls)):
                if got == SHAPE:
                    assert need == "0"
                    continue
                assert got.startswith("0 "), (calls[into], got)
                run = launches(got)
                if run[0][0] == "embedding_few_kernel":
                    assert need == "0" and len(run) == 1
                    continue
                assert ask([f"embedding_bwd {n} {vocab} {d} {bf16} {into} {int(need) - 1}"]) == [WS]
                sums = [(a, w) for k, a, w in run if k == "embedding_sum_kernel"]
                piece = int(sums[0][0].split(",")[1])
                pieces = -(-n // piece)
                blocks = -(-(d * (2 if bf16 else 4) // 16) // 64)
                assert len(sums) == 1 and -(-pieces * blocks // 4) <= sums[0][1] <= -(-(pieces * blocks + vocab) // 4)
                part = pieces * 2 * d * 4 if pieces > 1 else 0
                counts = [w for k, _, w in run if k == "embedding_count_kernel"]
                if not counts:
                    assert run[0][0] == "embedding_gather_kernel" and int(need) >= n * 8 + vocab + part
                elif into:                               # every workgroup sorts
                    digits = len(counts)
                    bits = -(-(vocab.bit_length()) // digits)
                    assert bits <= 9 and max(counts) <= 128 and int(need) >= 2 * n * 8 + vocab + max(counts) * (4 << bits) + part
                assert ([k for k, _, _ in run if k == "embedding_join_kernel"] != []) == (pieces > 1)


def test_an_embedding_takes_every_shape_below_its_documented_limits(ask):
    for bf16, unit in ((0, 4), (1, 8)):
        for n, d in (((1 << 26) - 1, 64 * unit), (1 << 26, 64 * unit), ((1 << 24) - 1, 1 << 20), (1 << 24, 1 << 20), (2 ** 31 - 1, unit), (2 ** 31 - 1, 2 * unit),
                     (1 << 30, 4 * unit), (1 << 30, 3 * unit), ((1 << 30) - 64, 3 * unit)):
            threads = 1
            while threads < d // unit and threads < 256:
                threads *= 2
            got, = ask([f"lookup {n} 100 {d} {bf16}"])
            assert bool(launches(got)) if n * threads < (1 << 32) - 256 else got == SHAPE, (n, d, got)
        for n, vocab, d in ((1 << 30, 1000, unit), ((1 << 30) + 1, 1000, unit), (100, (1 << 26) - 1, unit), (100, (1 << 26) - 4, unit), (1, 1 << 26, unit),
                            (1 << 20, 1000, 1 << 20), (1 << 16, 1000, 1 << 20), (1 << 17, 1000, 1 << 20), (1 << 30, 1 << 25, 64 * unit),
                            (1 << 30, (1 << 25) - 1, 64 * unit), (2 ** 31 - 1, 2 ** 31 - 1, 1 << 20)):
            blocks = -(-d // (64 * unit))
            pieces = -(-n // (32 if n // 32 * blocks >= 1024 else 8))
            fits = n <= 1 << 30 and pieces * blocks + vocab < 1 << 26 and -(-pieces // 16) * -(-d // 256) < 1 << 22
            need, = ask([f"embedding_bwd_bytes {n} {vocab} {d} {bf16}"])
            for into in (0, 1):
                got, = ask([f"embedding_bwd {n} {vocab} {d} {bf16} {into} {need}"])
                assert bool(launches(got)) if fits else (got, need) == (SHAPE, "0"), (n, vocab, d, into, got)


def test_the_scratch_of_a_layer_norm_s_gradients_holds_their_parts(ask):
    """A workgroup of the main launch writes two rows of d_model numbers, unless it is the only one."""
    for d in (8, 64, 512, 1032, 2048, 2560, 4096, 5120, 8192):
        for rows in (1, 2, 3, 100, 4095, 4096, 65536, 1 << 25):
            need = int(ask([f"norm_bwd_bytes {rows} {d}"])[0])
            if need == 0:
                assert ask([f"norm {rows} {d} 1 1", f"norm_bwd {rows} {d} 1 1 1000000000"]) == [SHAPE, SHAPE]
                continue
            for resid in (0, 1):
                for bias in (0, 1):
                    got, less = ask([f"norm_bwd {rows} {d} {resid} {bias} {need}", f"norm_bwd {rows} {d} {resid} {bias} {need - 1}"])
                    run = launches(got)
                    assert less == WS and run[0][0] == "layernorm_residual_bwd_kernel" and need >= run[0][2] * 2 * d * 4, (rows, d, got)
                    assert [k for k, _, _ in run[1:]] == (["layernorm_dweight_kernel"] if run[0][2] > 1 else []), (rows, d, got)
                    assert launches(ask([f"norm {rows} {d} {resid} {bias}"])[0])


@pytest.mark.parametrize("bf16", [0, 1])
def test_the_scratch_of_log_probabilities_holds_what_the_parts_of_rows_write(ask, bf16):
    """A part of a row leaves its maximum, two sums and its alternatives, 8 bytes each, unless it is the whole row."""
    for rows in (1, 3, 7, 100, 512, 1023, 1024, 5000, (1 << 24) - 1):
        for vocab in (1, 2, 63, 1000, 4096, 50001, 262144, (1 << 30) - 1):
            for top in (0, 1, 5, 64):
                if top > vocab:
                    continue
                need, = ask([f"logprobs_bytes {rows} {vocab} {top} {bf16}"])
                for entropy in (0, 1):
                    got, = ask([f"logprobs {rows} {vocab} {vocab + 3} {top} {bf16} {entropy} {need}"])
                    cut = -(-vocab // (4096 if bf16 else 2048))
                    if rows * cut >= 1 << 24:
                        assert (got, need) == (SHAPE, "0")
                        assert ask([f"logprobs_bwd {rows} {vocab} {vocab + 3} {bf16} {entropy}"]) == [SHAPE]
                        continue
                    run = launches(got)
                    parts = run[0][2] // rows
                    assert run[0][0] == "token_logprobs_kernel" and run[0][2] == rows * parts and run[0][2] <= max(rows, 1024), got
                    if parts == 1:
                        assert need == "0" and len(run) == 1
                    else:
                        assert [(k, w) for k, _, w in run[1:]] == [("token_logprobs_join_kernel", rows)]
                        assert int(need) >= run[0][2] * (12 + 8 * top)
                        assert ask([f"logprobs {rows} {vocab} {vocab} {top} {bf16} {entropy} {int(need) - 1}"]) == [WS]
                    grad = launches(ask([f"logprobs_bwd {rows} {vocab} {vocab + 3} {bf16} {entropy}"])[0])
                    assert [(k, w) for k, _, w in grad] == [("token_logprobs_bwd_kernel", rows * cut)]
