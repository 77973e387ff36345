"""The row kernels are built in the variants that some call reaches, and in no
other: the rules of residual_norm.cu restated over all widths."""
import pathlib
import re

from wide_compiler import ops

SRC = (pathlib.Path(ops.__file__).resolve().parents[1] / "csrc" / "residual_norm.cu").read_text()
BLOCK = 512


def team(d, k):
    if d <= 32 * k:
        return "WARP"
    return "BLOCK" if -(-d // (32 * k)) * 32 <= BLOCK else "PAIR"


def body(of, name):
    text = SRC[SRC.index("struct " + of):]
    text = text[text.index(name):]
    return text[:text.index("\n    }\n")]


def test_forward_teams():
    reached = set()
    for d in range(1, 8193):
        for ve in (1, 2, 4, 8):
            if d % ve == 0:
                for many in (False, True):
                    k = 16 if ve >= 4 and (d > 4096 or many) else 8
                    reached.add((min(ve, 4), k, team(d, k)))
    assert {v for v, k, t in reached if t == "PAIR"} == {1, 2}
    assert all((v, 8, t) in reached for v in (1, 2, 4) for t in ("WARP", "BLOCK"))
    assert (4, 16, "WARP") in reached and (4, 16, "BLOCK") in reached
    rule = body("ForwardLaunch", "int team()")
    assert re.search(r"if constexpr \(VE < 4\)[^;]*PAIR", rule) and rule.count(", PAIR, ") == 2


def test_quantize_teams():
    reached = set()
    for d in range(1, 32 * BLOCK + 1):
        for ve in (1, 2):
            most = 16 if ve == 1 else 32
            if d % ve == 0 and d <= most * BLOCK:
                for many in (False, True):
                    k = 8 if d <= 8 * BLOCK and (d <= 256 or not many) else 16 if d <= 2048 else most
                    reached.add((ve, k, team(d, k)))
    assert reached == {(v, k, t) for v in (1, 2) for k in (8, 16) for t in ("WARP", "BLOCK")} | {(2, 32, "BLOCK")}
    assert re.search(r"if constexpr \(K <= 16\)[^;]*WARP", body("QuantizeLaunch", "int team()"))
