"""Which attention kernel a call takes (no GPU): the rule of csrc/kv4_attention.cuh, compiled for the host, against its
restatement in kv4_exact.py, which the GPU tests go by; and the calls that are meant for the kernel for many query rows."""
import os
import random
import re
import subprocess

from kv4_exact import many_rows

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def rule(tmp_path, cases):
    with open(os.path.join(ROOT, "unpopped_b200", "csrc", "kv4_attention.cuh")) as f:
        text = re.search(r"inline bool many_rows\(.*?\n}\n", f.read(), re.S).group(0)
    src, exe = tmp_path / "rule.cpp", tmp_path / "rule"
    src.write_text("#include <cstdint>\n#include <cstdio>\n" + text +
                   "int main() { long long r, p, d, s; while (scanf(\"%lld %lld %lld %lld\", &r, &p, &d, &s) == 4)"
                   " puts(many_rows(r, p, d, s) ? \"1\" : \"0\"); }\n")
    subprocess.run(["g++", "-o", str(exe), str(src)], check=True)
    given = "".join(f"{r} {p} {d} {s}\n" for r, p, d, s in cases)
    return [line == "1" for line in subprocess.run([str(exe)], input=given, capture_output=True, text=True).stdout.split()]


def test_the_tests_rule_is_the_kernels(tmp_path):
    rng = random.Random(4)
    calls = []
    for _ in range(3000):
        tokens, batch, kv = int(2 ** rng.uniform(0, 16)), int(2 ** rng.uniform(0, 8)), int(2 ** rng.uniform(0, 5))
        calls.append((tokens, batch, kv * rng.randint(1, 100), kv, rng.choice([32, 64, 96, 128, 256]), rng.choice([148, 132, 1])))
    want = rule(tmp_path, [(-(-t // b) * (h // kv), b * kv, d, s) for t, b, h, kv, d, s in calls])
    assert [many_rows(*c) for c in calls] == want and 100 < sum(want) < 2900


def test_the_smoke_test_runs_both_kernels():
    """One sequence of 40 tokens, a key/value head of 64: 2 query heads and one token, and 400 heads."""
    with open(os.path.join(ROOT, "__graft_entry__.py")) as f:
        text = f.read()
    heads = 2 * int(re.search(r"kv4_attention\(qr\.repeat\(1, (\d+), 1\)", text).group(1))
    assert many_rows(40, 1, heads, 1, 64) and not many_rows(1, 1, 2, 1, 64)
