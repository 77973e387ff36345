"""Index arithmetic of the block-boundary kernels at the largest sizes that
their entry points take, on the CPU: the expressions are read from the kernel
sources and compiled for the host, where an overflow of signed numbers ends
the program."""
import pathlib
import re
import shutil
import subprocess

import pytest

from wide_compiler import ops

CSRC = pathlib.Path(ops.__file__).resolve().parents[1] / "csrc"
MOST = 0x7fffffff                       # rows of a call


def source(name):
    return (CSRC / name).read_text()


def run_on_host(tmp_path, body):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(body)
    for cmd in (["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", str(src), "-o", str(exe)],
                [str(exe)]):
        p = subprocess.run(cmd, capture_output=True, text=True)
        assert p.returncode == 0, p.stdout + p.stderr


@pytest.mark.parametrize("name, kernel", [("residual_norm.cu", "forward_kernel"), ("residual_norm.cu", "quantize_kernel"),
                                          ("residual_norm_bwd.cuh", "backward_kernel")])
def test_rows_ahead_of_the_last_ones(name, kernel, tmp_path):
    """A walk asks for the rows ahead of it; at the end of 2^31 - 1 rows there are none."""
    text = source(name)
    text = text[text.index(kernel + "("):]
    text = text[:text.index("\n}\n")]
    params, guard = re.search(r"auto fetch = \[&\]\(int stage, (.*?)\) \{\s*if \((.*)\)[ {]", text).groups()
    calls = [c.split(",", 1)[1] for c in re.findall(r"\bfetch\((.*)\);", text) if "ring.fetch(" + c not in text]
    assert len(calls) >= 3
    walk = re.search(r"struct Walk \{.*?\n\};", source("residual_norm.cuh"), re.S).group(0)
    checks = "".join(f"""
        for (int row = walk.first; row < walk.end; ++row)
            for (int k = 0; k < ring.AHEAD; ++k)
                if (holds({c}) != ((int64_t){c.strip().replace(",", " +")} < walk.end)) return 3;""" for c in calls)
    run_on_host(tmp_path, f"""
#include <cstdint>
#define __device__
#define __forceinline__ inline
{walk}
int main() {{
    struct {{ int STAGES = 3, AHEAD = 2; }} ring;
    const int teams = 1 << 24;
    for (int t = 0; t < teams; t += teams - 1) {{
        const Walk walk(t, teams, {MOST});
        if (walk.end <= walk.first || (t > 0 && walk.end != {MOST})) return 2;
        auto holds = [&]({params}) {{ return {guard}; }};{checks}
    }}
    return 0;
}}
""")


def test_places_of_the_longest_row(tmp_path):
    """Rows that a block takes at 1024 values a turn: no turn past the end, up to the longest row of
    single values."""
    text = source("residual_norm.cu")
    longest = int(re.search(r"d > (0x[0-9a-f]+)\)", text[text.index("int widek_quantize_rows_fwd("):]).group(1), 16)
    kernel = text[text.index("quantize_long_kernel("):]
    loops = re.findall(r"for \((.* c = .*?)\) (?:top|put)", kernel[:kernel.index("\n}\n")])
    assert len(loops) == 2
    turns = "".join(f"""
        {{
            int64_t n = 0;
            for ({loop}) if (c < 0 || c >= {longest} || ++n > {-(-longest // 1024)}) return 3;
            if (n < {longest // 1024}) return 4;
        }}""" for loop in loops)
    run_on_host(tmp_path, f"""
#include <cstdint>
int main() {{
    const int nvec = {longest};
    for (int t = 0; t < 1024; t += 1023) {{
        struct {{ int t, threads; }} at{{t, 1024}};{turns}
    }}
    return 0;
}}
""")
