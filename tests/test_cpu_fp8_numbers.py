"""What the attention over 8-bit pages multiplies with in place of a weight and of a query (pie_chunk_attn.cuh), over all numbers there are, against what is said of it: the kernel's own constants, the
documented bounds."""
import os
import re

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def text(*path):
    with open(os.path.join(ROOT, *path)) as f:
        return f.read()


KERNEL = text("proxy_inference_engine_b200", "csrc", "pie_chunk_attn.cuh")


def thirds(x):
    """chunk_thirds of fp16 numbers, each with its half of a register to itself."""
    add, keep = (int(g, 16) for g in re.search(r"to\[i\] = \(x \+ 0x(\w{4})0080u\) & 0x(\w{4})ff00u;", KERNEL).groups())
    parts = []
    for _ in range(3):
        parts.append(((x.view(np.uint16).astype(np.uint32) + add) & keep).astype(np.uint16).view(np.float16))
        x = (x.astype(np.float64) - parts[-1].astype(np.float64)).astype(np.float16)
    return parts


def documented():
    """Of a weight, and of the row's largest; of a row's largest query: exponents of two, in either place."""
    got = set()
    for where in (text("include", "pie_b200.h"), text("proxy_inference_engine_b200", "ops.py")):
        where = " ".join(where.replace("*", " ").split())
        weight = re.search(r"fp16, off by (?:up to )?2\^-(\d+) of one and (?:by )?2\^-(\d+) of the row's largest", where)
        query = re.search(r"of (?:their |the )?queries what is 2\^-(\d+) of the row's largest is lost", where)
        got.add((*weight.groups(), query and query.group(1)))
    assert len(got) == 1
    return [int(n) for n in got.pop()]


def test_weights_in_three_numbers():
    """Of a row's largest weight, 2^9 at least, and of one's own: the largest error over all weights there are, which are fp16's numbers and what lies between them."""
    above, units = (float(g) for g in re.search(r"const float m = move \? now \+ (\d)\.f : was;[\s\S]{0,300}?\? 0\.f : (\d+)\.f - m;", KERNEL).groups())
    least = 2.0 ** (units - above)
    ceiling = float(re.search(r"over = mx > (\d+)\.f;", KERNEL).group(1))
    of_one, of_largest, _ = documented()
    x = np.arange(np.float16(2.0 ** ceiling).view(np.uint16) + 1, dtype=np.uint16).view(np.float16)
    parts = thirds(x)
    for p in parts:   # e5m2 is fp16's upper byte
        assert not (p.view(np.uint16) & 0xff).any() and np.isfinite(p.astype(np.float64)).all()
    split = sum(p.astype(np.float64) for p in parts)
    x = x.astype(np.float64)
    assert split[np.abs(x) >= 2.0 ** -5].tolist() == x[np.abs(x) >= 2.0 ** -5].tolist()
    # weights next to a number, up to half of the way to its neighbours
    half = np.diff(x) / 2
    worst = np.maximum(np.abs(split[:-1] - (x[:-1] + half)), np.abs(split[1:] - (x[1:] - half)))
    own = 2.0 ** -of_one * (x[:-1] + half)
    assert (worst - own).max() <= 2.0 ** -of_largest * least * (1 + 2.0 ** -8)
    # and no smaller power of two would do
    assert (worst - own).max() > 2.0 ** -(of_largest + 1) * least * (1 + 2.0 ** -8)
    assert (worst > 2.0 ** -(of_one + 1) * (x[:-1] + half) * (1 + 2.0 ** -8) + 2.0 ** -of_largest * least).any()


def test_queries_in_two_numbers():
    """Features of a row whose largest lies at 2^7 .. 2^8."""
    v = torch.arange(0x4380, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).float()   # (up to 256)
    first = v.to(torch.float8_e4m3fn).float()
    both = (first + (v - first).to(torch.float8_e4m3fn).float()).double()
    off = (both - v.double()).abs()
    query = documented()[2]
    assert float(off.max()) <= 2.0 ** -query * 2.0 ** 7 and float(off.max()) > 2.0 ** -(query + 1) * 2.0 ** 7
    assert not off[v >= 2.0 ** -2].any()
