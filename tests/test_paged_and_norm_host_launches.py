"""What the host code of the paged and RMS norm entry points decides, on the CPU: as tests/test_host_launches.py, every signed overflow an
abort, launches recorded instead of made (tests/host_launches)."""
import os
import re
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from tests.test_host_launches import CHECKED, ROOT

NULL, SHAPE, MISAL, WS = "-1", "-2", "-4", "-5"


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("host")

    def compile_(name):
        obj = str(tmp / (name + ".o"))
        subprocess.check_call(["/opt/rocm/bin/hipcc", "--offload-arch=gfx950", "--offload-host-only", "-O1", "-std=c++17", "-w", *CHECKED, "-c",
                               os.path.join(ROOT, "tyr_amd", "csrc", name + ".hip"), "-o", obj])
        return obj
    with ThreadPoolExecutor() as pool:
        objs = list(pool.map(compile_, ("capi", "paged", "rmsnorm")))
    main, exe = str(tmp / "recorder.o"), str(tmp / "recorder")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-D__HIP_PLATFORM_AMD__=1", "-isystem", "/opt/rocm/include", "-c",
                           os.path.join(ROOT, "tests", "host_launches", "paged_recorder.cpp"), "-o", main])
    # what the other kernel files and the fat binaries would define is never reached
    subprocess.check_call(["/opt/rocm/llvm/bin/clang++", main, *objs, "-fsanitize=signed-integer-overflow", "-fsanitize-minimal-runtime",
                           "-Wl,--unresolved-symbols=ignore-all", "-o", exe])

    def run(lines):
        r = subprocess.run([exe], input="\n".join(lines) + "\n", capture_output=True, text=True)
        got = r.stdout.splitlines()
        assert r.returncode == 0 and len(got) == len(lines), (lines[min(len(got), len(lines) - 1)], r.returncode, r.stderr[-300:])
        return got
    return run


def test_the_scratch_query_knows_the_shapes_that_a_call_refuses(ask):
    """It overflowed for some and asked for terabytes; callers allocate by it before the call can refuse."""
    shapes = [(1, 2147483633, 1, 128, 16, 100), (1, 2147483632, 1, 128, 16, 100), (1, 2 ** 31 - 1, 1, 64, 16, 1), (1, 1 << 26, 1, 64, 16, 1),
              (1 << 26, 1, 1, 64, 16, 1), (2 ** 31 - 1, 1, 1, 128, 16, 1), (1 << 16, 1, 1, 128, 16, 1 << 15), (1, 1, 1, 128, 16, (1 << 27) - 1),
              (16, 1, 1, 128, 16, (1 << 27) - 1), (1 << 25, 1, 1, 128, 16, 60), (1 << 12, 1 << 13, 1, 64, 16, 1 << 12), (3, 34, 2, 64, 48, 999)]
    for s in shapes:
        need, = ask([f"decode_bytes {' '.join(map(str, s))}"])
        for e4m3 in (0, 1):
            with_it, = ask([f"decode {' '.join(map(str, s))} 0 0 {e4m3} {int(need) or 1 << 50}"])
            if with_it.startswith("0 "):
                assert int(need) <= 1 << 33 and (int(need) == 0 or ask([f"decode {' '.join(map(str, s))} 0 0 {e4m3} {int(need) - 1}"]) == [WS])
            else:
                assert (with_it, need) == (SHAPE, "0"), s


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (8, 2), (17, 1), (32, 1), (33, 1), (66, 2), (128, 1), (130, 1), (1200, 600)])
def test_the_scratch_of_a_decode_holds_what_any_window_writes(ask, Hq, Hkv, D):
    """The query knows neither the window nor the pages' format.  A launch of shares has one workgroup more than there are; a wave writes
    at most two partial results of each of its query heads: D numbers, a maximum and a sum."""
    G = Hq // Hkv
    for B in (1, 3, 70, 2000):
        for page, width in ((16, 1), (16, 16), (16, 17), (48, 30), (256, 40), (64, 2000)):
            shape = f"{B} {Hq} {Hkv} {D} {page} {width}"
            need, = ask([f"decode_bytes {shape}"])
            calls = [f"decode {shape} {window} {sinks} {e4m3} {need}" for window in (0, 1, 100, 225, 1000, 1 << 40) for sinks in (0, 4, 300, 1 << 40)
                     for e4m3 in (0, 1)]
            for call, got in zip(calls, ask(calls)):
                if got == SHAPE:                         # too many steps, whatever the window
                    assert need == "0"
                    continue
                m = re.fullmatch(r"0 paged_decode_kernel<\d+,(?:true|false),(\d),(true|false)>:(\d+)( paged_join\w*<\d+>:\d+)?", got)
                assert m, (call, got)
                if m[4]:
                    beside = -(-G // 16) if m[2] == "true" else 1
                    waves = (int(m[3]) - 1) * beside
                    assert int(need) >= 8 * (B + 1) + waves * 2 * min(G, 16 * int(m[1])) * (D + 2) * 4, (call, got)


def test_a_decode_takes_every_shape_below_its_documented_limits(ask):
    """B Hq < 2^26, and steps of 32 rows of all heads (blocks of 16 query heads) < 2^30: the rest is refused."""
    for B, Hq, Hkv, page, width in ((1 << 25, 1, 1, 16, 60), (1 << 25, 1, 1, 16, 63), (1 << 25, 1, 1, 16, 62), (1 << 25, 2, 1, 16, 1), ((1 << 26) - 1, 1, 1, 16, 1),
                                    (1 << 26, 1, 1, 16, 1), ((1 << 26) - 1, 1, 1, 16, 31), (1 << 16, 1, 1, 16, 1 << 15), ((1 << 16) - 1, 1, 1, 16, 1 << 15),
                                    (15, 1, 1, 16, (1 << 27) - 1), (16, 1, 1, 16, (1 << 27) - 1), (15, 16, 1, 16, (1 << 27) - 1), (15, 17, 1, 16, (1 << 27) - 1),
                                    (1, (1 << 26) - 1, 1, 16, 16), (7, 170, 17, 48, 1000)):
        fits = B * Hq < 1 << 26 and B * Hkv * -(-(Hq // Hkv) // 16) * -(-page * width // 32) < 1 << 30
        for D in (64, 128):
            shape = f"{B} {Hq} {Hkv} {D} {page} {width}"
            need, = ask([f"decode_bytes {shape}"])
            for e4m3 in (0, 1):
                got, = ask([f"decode {shape} 0 0 {e4m3} {need}"])
                assert got.startswith("0 paged_decode_kernel") if fits else (got, need) == (SHAPE, "0"), (shape, got)


def test_row_scales_of_a_bf16_norm_are_not_looked_at(ask):
    for residual in (0, 1):
        assert ask([f"norm 4 64 {residual} 0 {at}" for at in (0, 2, 4096)]) == ask([f"norm 4 64 {residual} 0 0"]) * 3
        assert ask([f"norm 4 64 {residual} 0 2"])[0].startswith("0 rmsnorm_residual_kernel")
        assert ask([f"norm 4 64 {residual} 1 {at}" for at in (0, 2)]) == [NULL, MISAL]


def test_the_scratch_of_a_norm_s_gradients_holds_their_parts(ask):
    """A workgroup of the main launch writes a row of d_model numbers for dweight, unless it is the only one."""
    for d in (8, 64, 512, 1032, 2048, 2560, 4096, 5120, 8192, 16384):
        for rows in (1, 2, 3, 100, 4095, 4096, 65536, 2 ** 31 - 1):
            need = int(ask([f"norm_bwd_bytes {rows} {d}"])[0])
            for resid in (0, 1):
                got, less = ask([f"norm_bwd {rows} {d} {resid} {need}", f"norm_bwd {rows} {d} {resid} {need - 1}"])
                m = re.fullmatch(r"0 rmsnorm_residual_bwd_kernel<.*>:(\d+)( rmsnorm_dweight_kernel:\d+)?", got)
                assert m and less == WS and need >= int(m[1]) * d * 4 and (m[2] is None) == (m[1] == "1"), (rows, d, got)
