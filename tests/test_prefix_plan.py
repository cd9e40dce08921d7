"""How the attention of a shared prefix is cut (compiled for the host), and what its kernels and the softmax's do once a bounded wait has run out (read
from their sources: no wait is made to run out on a GPU)."""
import os
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llama.cu_b200", "csrc")
SMS = 148

MAIN = r"""
#include <cstdio>
#include "prefix_plan.hpp"
int main() {
    int n, group, nkvh, sms, dh;
    unsigned len;
    long long own;
    while (scanf("%d %d %d %u %d %d %lld", &n, &group, &nkvh, &len, &sms, &dh, &own) == 7) {
        const lcu::PrefixPlan p = lcu::prefix_plan(n, group, nkvh, len, sms, dh, own);
        printf("%d %d %d %d %d %d %d %zu %zu %zu", p.pairs, p.units, p.per, p.ctas, p.key_tiles, p.slot_rows, p.own_parts, lcu::prefix_own_row(p),
               lcu::prefix_ml_bytes(p, nkvh) + lcu::prefix_part_rows(p, nkvh) * dh * 4, lcu::prefix_bytes(n, group, nkvh, len, sms, dh));
        bool dealt = p.unit_at(0) == 0 && p.unit_at(p.ctas * p.per) == p.units;
        for (long long c = 0, pair = 0; c < p.ctas; ++c) {  // every CTA has units, all of them its own, and none is left out
            const long long u0 = p.unit_at(c * p.per), u1 = p.unit_at((c + 1) * p.per);
            dealt = dealt && u0 < u1;
            for (long long u = u0; u < u1 && p.units < 100000; u = (pair + 1) * p.key_tiles < u1 ? (pair + 1) * p.key_tiles : u1) {
                pair = u / p.key_tiles;
                const long long end = (pair + 1) * p.key_tiles < u1 ? (pair + 1) * p.key_tiles : u1;
                dealt = dealt && p.first_cta(pair) <= c && c <= p.last_cta(pair) && p.ahead(pair, u - pair * p.key_tiles) / p.per == c &&
                        p.ahead(pair, end - 1 - pair * p.key_tiles) / p.per == c;
            }
        }
        const long long show = p.pairs < 5000 ? p.pairs : 5000;
        for (long long i = 0; i < show; ++i) printf(" %d %d", p.first_cta(i), p.last_cta(i));
        printf(" %d %d %d %d\n", dealt, p.cost, lcu::prefix_walk(n, group, nkvh, len, own, sms, dh), lcu::own_splits((long long)n * nkvh, own + len, sms));
    }
}
"""

SHAPES = [(n, group, nkvh, length, dh, own) for n in (1, 2, 3, 16, 33, 80, 256, 1000) for group, nkvh in ((1, 1), (4, 8), (8, 8), (16, 2), (1, 32), (3, 5))
          for length in (1, 100, 128, 129, 2000, 8001, 32000) for dh, own in ((64, 0), (128, 2000), (128, 400000))]


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    d = tmp_path_factory.mktemp("prefix")
    (d / "main.cpp").write_text(MAIN)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC, str(d / "main.cpp"), "-o", str(d / "main")], check=True)

    def run(shapes):
        text = "\n".join(f"{n} {g} {h} {length} {SMS} {dh} {own}" for n, g, h, length, dh, own in shapes)
        out = subprocess.run([str(d / "main")], input=text, capture_output=True, text=True, check=True).stdout.strip().split("\n")
        return [list(map(int, line.split())) for line in out]
    return run


def test_every_unit_belongs_to_one_cta_and_every_piece_has_a_slot(plans):
    for shape, p in zip(SHAPES, plans(SHAPES)):
        n, group, nkvh, length, _, _ = shape
        pairs, units, per, ctas, key_tiles, slot_rows, parts, own_row, used, bound = p[:10]
        ends = list(zip(p[10:-4:2], p[11:-4:2]))
        assert key_tiles == -(-length // 128) and pairs == nkvh * -(-n * group // 256) and units == pairs * key_tiles, shape
        assert 1 <= ctas <= SMS and p[-4] == 1, shape
        last = n * group - (n * group - 1) // 256 * 256
        cost, cost_last = (3, 2) if n * group > 256 and last <= 128 else (1, 1)
        assert p[-3] == cost
        starts, at = [], 0
        for pair in range(len(ends)):
            starts.append(at)
            at += key_tiles * (cost_last if (pair + 1) % (pairs // nkvh) == 0 else cost)
        slots = set()
        for pair, (first, last) in enumerate(ends):
            end = starts[pair + 1] if pair + 1 < len(starts) else at
            assert first == starts[pair] // per and starts[pair] // per <= last <= (end - 1) // per, shape
            for cta in range(first, last + 1):
                assert cta + pair not in slots, shape
                slots.add(cta + pair)
        assert max(slots) < ctas + pairs and own_row == (ctas + pairs) * slot_rows and slot_rows == min(n * group, 256), shape
        assert used <= bound, shape


def test_parts_of_own_slots(plans):
    for shape, p in zip(SHAPES, plans(SHAPES)):
        blocks, parts = shape[0] * shape[2], p[6]
        assert (parts == 0 and blocks <= SMS) or (1 <= parts <= 8 and (parts == 1 or parts * blocks <= 3 * SMS)), shape
        if blocks <= SMS and shape[3] <= 128:
            assert (parts == 0) == (shape[1] <= 13), shape  # few parts to a row: as long as a block has few rows


def test_the_largest_call(plans):
    """2^28 units: costs of 3 each still fit."""
    for shape in [(4096, 16, 256, 128 * 4096, 128, 0), (4100, 16, 8, 128 * 130500, 128, 0), (65535, 16, 65535, 1, 128, 0)]:
        p = plans([shape])[0]
        assert p[1] <= 2 ** 28 < 2 * p[1] and p[-4] == 1 and 1 <= p[3] <= SMS


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_no_wait_of_these_kernels_is_endless():
    for name in ("prefix.cu", "verify.cu", "paged.cu"):
        text = source(name)
        assert "try_wait" not in text and "test_wait" not in text and "while (true)" not in text and "for (;;)" not in text  # the bounded ones of tc.cuh alone
        for wait in re.finditer(r"tc_(?:mbar|warp)_wait\(", text):
            line = text[text.rfind("\n", 0, wait.start()) + 1:wait.start()]
            assert re.search(r"(ok|here) = |&& *$|return ", line), line  # ... and what they answer is looked at


def test_the_prefix_kernel_leaves_after_its_copies_and_products_and_marks_its_rows():
    text = source("prefix.cu")
    body = text[text.index("prefix_tc_kernel(const PrefixArgs"):text.index("constexpr int OW_KEYS")]
    for load in re.finditer(r"at_ld32\(|tc_ld16\(", body):  # a warp loads an accumulator as a whole
        wait = body.rfind("tc_mbar_wait(", 0, load.start())
        assert "__all_sync" in body[wait:load.start()]
    leave = body[body.rindex("if (sh->abort_flag)"):body.index("tcgen05.dealloc")]
    assert leave.count("tc_warp_drain_ring(") == 2 and "tc_warp_commit(tc_smem(&sh->drain))" in leave and "0x7fc00000" in leave
    assert body[:body.rindex("if (sh->abort_flag)")].rstrip().endswith("__syncthreads();")  # when no warp can give up any more
    assert body.count("++k_issued") == body.count("++v_issued") == 1


def test_a_softmax_whose_wait_ran_out_is_nan_and_leaves_after_its_copy():
    text = source("verify.cu")
    body = text[text.index("softmax_kernel(const SoftmaxArgs"):text.index("struct VerifyArgs")]
    assert "if (AHEAD && !here) keep[0] = nan" in body and re.search(r"if \(!exchange\(.*\)\) s = nan", body) and "!here ? nan" in body
    assert body.rstrip().endswith("}") and "if (abort_flag) tc_warp_drain(tc_smem(&bar)" in body


def test_a_prefix_is_read_by_the_blocks_of_the_own_slots_while_that_is_short(plans):
    def walks(n, length, group=4, nkvh=8, dh=128, own=100):
        return plans([(n, group, nkvh, length, dh, own)])[0][-2]
    for n, short, long in ((1, 2000, 4000), (8, 600, 1000), (33, 100, 300), (100, 100, 300)):  # both measured
        assert walks(n, short) and not walks(n, long), n
    for n in (1, 3, 8, 33, 100, 1000, 20000):  # once too long, always
        kinds = [walks(n, length) for length in (1, 8, 16, 100, 500, 1000, 2000, 4000, 8000, 32000, 2 ** 31 - 1)]
        assert kinds == sorted(kinds, reverse=True) and kinds[0] and not kinds[-1], n
    for n, length in ((30000, 8), (1500, 63), (1000, 127), (500, 255)):  # what the GPU's tests of short prefixes rely on
        assert not walks(n, length) and not walks(n, length, dh=64) and walks(6, length) and walks(6, length, dh=64)


def test_splits_of_own_slots(plans):
    for shape, p in zip(SHAPES, plans(SHAPES)):
        blocks, slots, splits = shape[0] * shape[2], shape[5] + shape[3], p[-1]
        assert splits in (1, 2, 4, 8) and (splits == 1 or (blocks * splits // 2 <= SMS and slots > 64 * (splits // 2))), shape
