"""The overlap rules of the row grids that a call reads and writes, against every byte (no device needed)."""
import os
import random
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r'''
#include <cstdio>
#include "gs_overlap.h"
int main() {
  long long v[11];
  while (std::scanf("%lld %lld %lld %lld %lld %lld %lld %lld %lld %lld %lld", v, v + 1, v + 2, v + 3, v + 4, v + 5, v + 6, v + 7, v + 8, v + 9, v + 10) == 11) {
    gs::RowGrid a{(std::uintptr_t)v[0], v[1], v[2], v[3], v[4], v[5]}, b{(std::uintptr_t)v[6], v[7], v[8], v[9], v[10], v[5]};
    std::printf("%d %d\n", gs::rows_overlap(a) ? 1 : 0, gs::rows_overlap(a, b) ? 1 : 0);
  }
}
'''


def spans(base, tokens, heads, token, head, row):
    return [(base + t * token + h * head, base + t * token + h * head + row) for t in range(tokens) for h in range(heads)]


def meet(a, b):
    return any(x0 < y1 and y0 < x1 for x0, x1 in a for y0, y1 in b)


def test_rules_against_every_pair_of_rows(tmp_path):
    src, exe = tmp_path / "overlap.cc", tmp_path / "overlap"
    src.write_text(SOURCE)
    inc = os.path.join(ROOT, "gemma-webgpu-engine_b200", "csrc")
    subprocess.run(["g++", "-std=c++17", "-I", inc, str(src), "-o", str(exe)], check=True)
    rng = random.Random(5)
    cases = []
    for _ in range(4000):
        row = rng.choice([1, 4, 16])
        tokens, heads = rng.randint(1, 6), rng.randint(1, 6)
        token, head = row + rng.randint(0, 12 * row), row + rng.randint(0, 12 * row)
        base, base2 = 1000 + rng.randint(0, 40 * row), 1000 + rng.randint(0, 40 * row)
        token2, head2 = (token, head) if rng.random() < 0.6 else (token, row + rng.randint(0, 3 * row)) if rng.random() < 0.6 else \
            (row + rng.randint(0, 12 * row), head)
        cases.append((base, tokens, heads, token, head, row, base2, tokens, heads, token2, head2))
    for _ in range(1000):  # slices of one buffer
        row, tokens, heads, heads2 = 4, rng.randint(2, 5), rng.randint(2, 4), rng.choice([4, 8])
        token = row * rng.randint(12, 24)
        cases.append((1000, tokens, heads, token, row, row, 1000 + row * rng.randint(0, 24), tokens, heads, token, heads2))
    text = "\n".join(" ".join(map(str, c)) for c in cases)
    got = [tuple(map(int, line.split())) for line in
           subprocess.run([str(exe)], input=text, capture_output=True, text=True, check=True).stdout.splitlines()]
    assert len(got) == len(cases)
    exact = beside = 0
    for c, (own, both) in zip(cases, got):
        base, tokens, heads, token, head, row, base2, _, _, token2, head2 = c
        a, b = spans(base, tokens, heads, token, head, row), spans(base2, tokens, heads, token2, head2, row)
        assert own == any(x[0] < y[1] and y[0] < x[1] for i, x in enumerate(a) for y in a[i + 1:])
        truth = meet(a, b)
        assert both or not truth
        if (tokens == 1 or token == token2) and (heads == 1 or head == head2):
            assert both == truth
            exact += 1
        elif tokens > 1 and token == token2:  # side by side in every token of one buffer
            r, ea, eb = (base2 - base) % token, (heads - 1) * head + row, (heads - 1) * head2 + row
            if r >= ea and r + eb <= token:
                assert not both
                beside += 1
    assert exact > 1000 and beside > 20


def test_wide_strides_do_not_wrap(tmp_path):
    src, exe = tmp_path / "overlap.cc", tmp_path / "overlap"
    src.write_text(SOURCE)
    inc = os.path.join(ROOT, "gemma-webgpu-engine_b200", "csrc")
    subprocess.run(["g++", "-std=c++17", "-I", inc, str(src), "-o", str(exe)], check=True)
    n, s = 2 ** 31 - 1, 2 ** 32 - 16
    text = f"{2**40} {n} 8 {s} 256 256 {2**41} {n} 8 {s} 256\n{2**40} {n} 8 {s} 256 256 {2**40 + 2048} {n} 8 {s} 256\n"
    out = subprocess.run([str(exe)], input=text, capture_output=True, text=True, check=True).stdout.split()
    assert out[0] == "0" and out[2] == "0" and out[3] == "0"
