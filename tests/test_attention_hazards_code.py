"""What the attention kernels' assembly has to keep by itself, read from the code
that the sources compile to (no GPU needed).

The compiler puts the waits that the hardware lacks between an instruction and
one that uses its result, but not before inline assembly:
* a maximum of matrix products (max3) reads registers that the products write
  some time after they were issued.  A chain of maxima starts from an instruction
  that the compiler knows; without it the maximum was of unfinished sums, other
  ones from call to call;
* a load into LDS takes its base from registers that a lane was read into.

Registers that are spilled must come back under a full mask: lanes masked at that
moment would hold something else (test_linear_code.py)."""
import os
import random
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
SOURCES = ("attn_tile", "attn_tile32", "attn_shared", "attn_forms")
# wait states from a product to an instruction that reads it: passes and 4, of
# 32-bit products passes and 2; from a lane's value in a scalar register to a
# load that uses it
PRODUCT = {"v_mfma_f32_32x32x16_f16": 8 + 4, "v_mfma_f32_32x32x16_bf16": 8 + 4,
           "v_mfma_f32_32x32x2_f32": 16 + 2}
BASE = 5


@pytest.fixture(scope="module")
def built(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    where, csrc = tmp_path_factory.mktemp("asm"), os.path.join(ROOT, "vectorstorekit_amd", "csrc")
    runs = [subprocess.Popen(
        [HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Xclang",
         "-target-feature", "-Xclang", "-packed-fp32-ops", "-I" + os.path.join(ROOT, "include"),
         "-I" + csrc, "--cuda-device-only", "-S", os.path.join(csrc, s + ".hip"), "-o",
         str(where / (s + ".s"))], stderr=subprocess.DEVNULL) for s in SOURCES]
    assert [r.wait(timeout=600) for r in runs] == [0] * len(runs)
    return {s: (where / (s + ".s")).read_text() for s in SOURCES}


class Kernel:
    """Its instructions (name, operands, written as assembly in the source?,
    comment), the labels' places and the ways to each."""

    def __init__(self, text):
        self.code, self.at, inline = [], {}, False
        for line in text.split("\n"):
            if "#ASM" in line:
                inline = "START" in line
            code, _, note = line.partition(";")
            label = re.match(r"(\.?\w+):", code.strip())
            if label:
                self.at[label[1]] = len(self.code)
            elif code.strip() and not code.strip().startswith("."):
                name, _, rest = code.strip().partition("\t" if "\t" in code.strip() else " ")
                rest = re.split(r",\s*(?![^\[]*\])", rest.strip())
                self.code.append((name, [x.split()[0] for x in rest if x], inline, note))
        self.ways = [[] for _ in range(len(self.code) + 1)]
        for i, (name, operands, _, _) in enumerate(self.code):
            if name.startswith(("s_branch", "s_cbranch")):
                self.ways[self.at[operands[0]]].append(i)
            if name not in ("s_branch", "s_endpgm", "s_setpc_b64"):
                self.ways[i + 1].append(i)

    def nearest(self, i, register, wrote, most):
        """Wait states, over every way to instruction i, since an instruction
        that wrote the register and for which wrote() is true: the smallest
        number of them, and the instruction's name."""
        seen, todo, found = {}, [(j, 0) for j in self.ways[i]], None
        while todo:
            j, waited = todo.pop()
            if waited >= most or seen.get(j, most) <= waited:
                continue
            seen[j] = waited
            name, operands, _, _ = self.code[j]
            if operands and register in registers(operands[0]) and not re.match(
                    r"s_cmp|s_cbranch|global_|ds_write|scratch_store|flat_store", name):
                if wrote(name) and (found is None or waited < found[0]):
                    found = waited, name
                continue
            step = int(operands[0]) + 1 if name == "s_nop" else 1
            todo += [(k, waited + step) for k in self.ways[j]]
        return found


def registers(operand):
    m = re.fullmatch(r"([vsa])\[(\d+):(\d+)\]", operand)
    if m:
        return {(m[1], i) for i in range(int(m[2]), int(m[3]) + 1)}
    m = re.fullmatch(r"([vsa])(\d+)", operand)
    return {(m[1], int(m[2]))} if m else set()


def kernels(text, pattern):
    for m in re.finditer(r"^(\S*" + pattern + r"\S*):\s.*?^\.Lfunc_end", text, re.M | re.S):
        yield m[1], Kernel(m[0])


@pytest.mark.parametrize("source,instances", [("attn_tile", 16), ("attn_tile32", 2),
                                              ("attn_shared", 6)])
def test_maxima_are_of_finished_products(built, source, instances):
    found = 0
    for name, k in kernels(built[source], "k_" + source + "I"):
        found += 1
        maxima = [i for i, x in enumerate(k.code) if x[2] and x[0] == "v_max3_f32"]
        assert len(maxima) >= 8, name
        for i in maxima:
            for r in set().union(*(registers(x) for x in k.code[i][1][1:])):
                near = k.nearest(i, r, lambda x: x.startswith("v_mfma"), 24)
                assert near is None or near[0] >= PRODUCT[near[1]], (name, k.code[i], near)
    assert found == instances


@pytest.mark.parametrize("source", SOURCES)
def test_loads_into_lds_have_their_base(built, source):
    found = 0
    for name, k in kernels(built[source], "k_" + source + "I"):
        for i, (what, operands, inline, _) in enumerate(k.code):
            if not inline or not what.startswith("global_load_lds"):
                continue
            found += 1
            for r in registers(operands[1]):
                near = k.nearest(i, r, lambda x: x.startswith("v_read"), BASE)
                assert near is None, (name, i, near)
    assert found


FULL = (1 << 64) - 1


def walk(k, seed, visits, steps=30000):
    """One way through the kernel, its comparisons decided at random (a scalar
    branch mostly for what was seen less often): reloads under a partial mask."""
    rng, partial = random.Random(seed), set()
    mask, scalar = {"exec": FULL}, None
    some = lambda: rng.choice((FULL, 0, rng.getrandbits(64), rng.getrandbits(64)))

    def value(x):
        if x in ("-1", "0"):
            return FULL if x == "-1" else 0
        key = x if x in ("exec", "vcc") else min(registers(x), default=None)
        return mask.setdefault(key, some()) if key else some()

    def put(x, v):
        for r in registers(x):
            mask.pop(r, None)
        mask[x if x in ("exec", "vcc") else min(registers(x))] = v & FULL

    i = 0
    for _ in range(steps):
        name, ops, _, note = k.code[i]
        visits[i] += 1
        if name == "s_endpgm":
            break
        if "Folded Reload" in note or name == "v_accvgpr_read_b32":
            if mask["exec"] != FULL:
                partial.add(i)
        saves = re.fullmatch(r"s_(and|or|andn2)_saveexec_b64", name)
        logic = re.fullmatch(r"s_(and|or|xor|andn2|orn2|not|mov)_b64", name)
        if name.startswith(("s_branch", "s_cbranch")):
            there, kind = k.at[ops[0]], name.rpartition("_")[2]
            if name == "s_branch":
                take = True
            elif kind[:4] in ("exec", "vccz", "vccn"):
                take = (value(kind[:-2] if kind.endswith("nz") else kind[:-1]) == 0) == (
                    not kind.endswith("nz"))
            else:
                if scalar is None:
                    take = visits[there] < visits[i + 1] if rng.random() < 0.8 else \
                        rng.random() < 0.5
                    scalar = take == (kind == "scc1")
                take = scalar == (kind == "scc1")
            i = there if take else i + 1
            continue
        if saves:
            a, e = value(ops[1]), mask["exec"]
            put(ops[0], e)
            put("exec", {"and": a & e, "or": a | e, "andn2": a & ~e}[saves[1]])
            scalar = mask["exec"] != 0
        elif logic:
            a, b = value(ops[1]), value(ops[2]) if len(ops) > 2 else 0
            put(ops[0], {"and": a & b, "or": a | b, "xor": a ^ b, "andn2": a & ~b,
                         "orn2": a | ~b, "not": ~a, "mov": a}[logic[1]])
            if logic[1] != "mov":
                scalar = value(ops[0]) != 0
        elif name == "s_cselect_b64":
            scalar = rng.random() < 0.5 if scalar is None else scalar
            put(ops[0], value(ops[1]) if scalar else value(ops[2]))
        elif name.startswith("v_cmp"):
            put(ops[0], some() & mask["exec"])
        elif name in ("s_cmp_eq_u64", "s_cmp_lg_u64") and ops[1] == "0":
            scalar = (value(ops[0]) == 0) == ("eq" in name)
        elif name.startswith(("s_cmp", "s_bitcmp")):
            scalar = None
        elif name.startswith(("s_", "v_read")) and ops:
            for r in registers(ops[0]):
                mask.pop(r, None)
            if not name.startswith(("s_mov", "s_load", "s_cselect", "s_mul", "s_nop", "s_wait",
                                    "v_read")):
                scalar = None
        i += 1
    return partial


@pytest.mark.parametrize("source,pattern,instances,walks", [
    ("attn_tile", r"k_attn_tileI\w+?Li256E", 4, 700), ("attn_tile", r"k_attn_tileI\w+?Li128E", 4, 5),
    ("attn_shared", "k_attn_sharedI", 6, 5),
    ("attn_forms", "k_attn_formsIDF16_Li8ELi1ELi1ELb1E", 1, 60)])
def test_spills_come_back_under_a_full_mask(built, source, pattern, instances, walks):
    """The kernels that have any (a head of 256 keeps its sums where others spill).
    Not looked at: operands that are not aligned, whose queries' words are built
    in memory, each read, changed and written back under one mask."""
    found = 0
    for name, k in kernels(built[source], pattern):
        found += 1
        back = {i for i, x in enumerate(k.code)
                if "Folded Reload" in x[3] or x[0] == "v_accvgpr_read_b32"}
        if not back:
            continue
        visits = [0] * (len(k.code) + 1)
        for seed in range(walks):
            assert not walk(k, seed, visits), (name, seed)
        assert sum(visits[i] > 0 for i in back) >= 0.9 * len(back), name
    assert found == instances
