"""The gated delta rule's built assembly: no result of a matrix product is read before it is there, on any path.

A product's result is not interlocked: instructions that read it have to come some wait states later, which the compiler
sees to.  Where an unrolled loop over products can end after each pass it was seen to count the way through all passes
and not the short one (`settle()` in delta_tiles.h stands against that).  Here every path behind every product is
walked, from an instruction to each of its successors, until its wait states have passed or its result is replaced.
The numbers are those that the compiler leaves between a product and its reader in straight code; a wait state is an
instruction, and s_nop n stands for n + 1."""
import concurrent.futures
import os
import re
import subprocess

import pytest

import build  # metal-drone-nav_amd/build.py

WAITS = {"v_mfma_f32_16x16x4_f32": 10, "v_mfma_f32_16x16x16_bf16": 8, "v_mfma_f32_16x16x32_bf16": 8}
SOURCES = ["delta_rule.hip", "delta_rule_backward.hip"]
REGISTER = re.compile(r"\b([va])(?:(\d+)\b|\[(\d+):(\d+)\])")
WITH_REGISTERS = ("v_", "ds_", "global_", "flat_", "buffer_", "scratch_")
READS_FIRST = ("v_cmp", "v_readlane", "v_readfirstlane", "v_permlane", "v_swap", "v_fmac", "v_dot2c",
               "ds_write", "global_store", "flat_store", "buffer_store", "scratch_store")
WRITES_NOTHING = ("v_cmp", "v_readlane", "v_readfirstlane", "ds_write", "global_store", "flat_store", "buffer_store",
                  "scratch_store")


def registers(text):
    found = set()
    for kind, one, first, last in REGISTER.findall(text):
        found |= {(kind, i) for i in range(int(one or first), int(one or last) + 1)}
    return frozenset(found)


def kernels(text):
    """name -> [(instruction, operands)], {label: place}"""
    for match in re.finditer(r"^(_Z\w+):\s*; @\1$(.*?)^\.Lfunc_end", text, re.S | re.M):
        code, labels = [], {}
        for line in match.group(2).split("\n"):
            line = line.split(";")[0].strip()
            if line.endswith(":"):
                labels[line[:-1]] = len(code)
            elif line and not line.startswith("."):
                name, _, rest = line.partition(" ")
                code.append((name, [x.strip() for x in re.split(r",\s*(?![^\[]*\])", rest)]))
        yield match.group(1), code, labels


def early_reads(code, labels):
    """(product, reader, wait states between them) of every result read too early."""
    def after(at):
        name, operands = code[at]
        if name == "s_endpgm":
            return []
        if name == "s_branch":
            return [labels[operands[0]]]
        return [at + 1] + ([labels[operands[0]]] if name.startswith("s_cbranch") else [])

    found = []
    for start, (name, operands) in enumerate(code):
        if not name.startswith("v_mfma"):
            continue
        seen, todo = {}, [(at, 0, registers(operands[0])) for at in after(start)]
        while todo:
            at, waited, live = todo.pop()
            if not live or waited >= WAITS[name] or seen.get((at, live), 99) <= waited:
                continue
            seen[at, live] = waited
            other, given = code[at]
            read = written = frozenset()
            if other.startswith("v_mfma"):  # (the last operand, what is added to, has a way of its own)
                read, written = registers(given[1]) | registers(given[2]), registers(given[0])
            elif other.startswith(WITH_REGISTERS):
                read = registers(" ".join(given if other.startswith(READS_FIRST) else given[1:]))
                written = frozenset() if other.startswith(WRITES_NOTHING) or not given else registers(given[0])
            if read & live:
                found.append((start, code[start], at, code[at], waited))
            passed = 1 + int(given[0], 0) if other == "s_nop" else 1
            todo += [(to, waited + passed, live - written) for to in after(at)]
    return found


def test_the_walk_finds_an_early_read():
    """A loop that can end after one product: the way out passes the reader five wait states later."""
    code = [("v_mfma_f32_16x16x32_bf16", ["v[0:3]", "v[4:7]", "v[8:11]", "v[0:3]"]), ("s_cbranch_scc1", ["out"]),
            ("s_nop", ["15"]), ("s_nop", ["3"]), ("v_add_f32_e32", ["v20", "v2", "v2"]), ("s_endpgm", [""])]
    assert [(f[2], f[4]) for f in early_reads(code, {"out": 3})] == [(4, 5)]
    assert not early_reads(code, {"out": 2})
    code[4] = ("v_add_f32_e32", ["v2", "v20", "v20"])
    assert not early_reads(code, {"out": 3})


def assembly(source):
    command = [build.HIPCC] + build.FLAGS + ["--cuda-device-only", "-S", os.path.join(build.HERE, "csrc", source), "-o", "-"]
    return subprocess.run(command, capture_output=True, text=True, check=True).stdout


@pytest.mark.skipif(not os.path.exists(build.HIPCC), reason="no hipcc")
def test_no_result_is_read_early():
    with concurrent.futures.ThreadPoolExecutor() as pool:
        texts = list(pool.map(assembly, SOURCES))
    count = 0
    for source, text in zip(SOURCES, texts):
        for name, code, labels in kernels(text):
            products = sum(i.startswith("v_mfma") for i, _ in code)
            count += products
            assert not products or not early_reads(code, labels), (source, name)
    assert count > 1000
