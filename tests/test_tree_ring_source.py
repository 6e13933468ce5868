"""The model of ``test_tree_ring`` is the kernel's: what it took over from ``tree_attention_sm100.cu`` by hand
stands in the source as it stands in the model.  A change to the kernel's barriers, ring or order of tiles
fails here until the model follows it."""
from __future__ import annotations

import inspect
import re
from pathlib import Path

from tests import test_tree_ring as model

SOURCE = (Path(__file__).resolve().parent.parent / "moeinfra_b200/csrc/tree_attention_sm100.cu").read_text()
CODE = re.sub(r"\s+", " ", re.sub(r"//[^\n]*", "", SOURCE))
MODEL = re.sub(r"\s+", " ", inspect.getsource(model.walk))


def _constant(name):
    return int(re.search(rf"constexpr int {name} = (\d+);", CODE).group(1))


def test_items_readers_and_stages():
    readers, ahead = re.search(r"readers, items_ahead = (\d+), (\d+)", MODEL).groups()
    assert (_constant("kReaders"), _constant("kItems")) == (int(readers), int(ahead))
    most = re.search(r"constexpr int kStages = (\d+) \* (\d+) / kHalves;", CODE).groups()
    stages = {int(most[0]) * int(most[1]) // (hd // 64) for hd in (64, 128)}
    marks = [m for m in model.test_every_wait_is_for_its_phase.pytestmark if m.name == "parametrize"]
    assert stages == set(marks[0].args[1])
    assert "constexpr int kThreads = 12 * 32;" in CODE and "Clock(seed, 12)" in MODEL


def test_arrivals_that_each_barrier_counts():
    counts = dict(re.findall(r"mbar_init\(saddr\(&s_(\w+)(?:\[\w+\])*\), (\w+)\);", CODE))
    assert len(counts) == len(re.findall(r"mbar_init\(", CODE))
    names = {"full": "full", "empty": "empty", "qfull": "q_full", "qempty": "q_empty", "done": "done",
             "read": "read", "itfull": "it_full", "itempty": "it_empty"}
    for theirs, ours in names.items():
        want = re.search(rf'bars\(\w+, (\w+), "{ours}"\)', MODEL).group(1)
        assert counts.pop(theirs) == {"readers": "kReaders"}.get(want, want), theirs
    pairs = re.search(r"for c, n in (\(\(.*?\)\))\)", MODEL).group(1)
    for count, name in re.findall(r'\((\d+), "(\w+)"\)', pairs):
        assert counts.pop(name.replace("_", "")) == count, name
    assert 'Bar(1, "tail")' in MODEL and counts.pop("tail") == "1"
    assert counts == {"drain": "1"}  # a warp's own, at its end


def test_the_order_of_the_ring():
    assert "int lead_of(bool two) { return two ? 1 : 2; }" in CODE
    assert (model.lead(True), model.lead(False)) == (1, 2)
    at = ("g + (is_v ? (i + lead < all ? 2 * i + lead + 1 : all + i) : i < lead ? i : 2 * i - lead)")
    assert at in CODE
    for two in (True, False):
        lead = model.lead(two)
        for n in range(1, 9):
            for i in range(n):
                assert model.place(True, i, n, two) == (2 * i + lead + 1 if i + lead < n else n + i)
                assert model.place(False, i, n, two) == (i if i < lead else 2 * i - lead)
    assert "is_k = j_k < all && (r <= lead || !(r - lead & 1))" in CODE
    assert "is_k = j_k < steps and (i <= lead(two) or (i - lead(two)) % 2 == 0)" in MODEL
    assert "mine = two ? all : (all + 1 - t) >> 1" in CODE and "return flags & 1 ? steps : (steps + 1 - t) >> 1;" in CODE
    assert MODEL.count("steps if two else (steps + 1 - t) >> 1") == 2


def test_who_waits_for_what():
    """The waits in the source, each with its phase, and where the next item is asked for."""
    for text in ("if (i == (is_v ? min(2, all - 1) : 0)) prepare();",
                 "warp_wait(saddr(&s_itfull[i]), n_it / kItems & 1, a.wait_ns)",
                 "warp_wait(saddr(&s_itempty[i]), (n_it / kItems & 1) ^ 1, a.wait_ns)",
                 "warp_wait(saddr(&s_pvdone[t][n & 1]), n >> 1 & 1, a.wait_ns)",
                 "warp_wait(saddr(&s_sfull[t][n_s & 1]), n_s >> 1 & 1, a.wait_ns)",
                 "if (i > 0) { if (!(ok = product_done(n_s - 1))) break;",
                 "if (ok && mine > 1) ok = product_done(n_s - 2); if (ok && mine > 0) ok = product_done(n_s - 1);",
                 "warp_wait(saddr(&s_done[pal]), n_pair & 1, a.wait_ns)",
                 "warp_wait(saddr(&s_read[pal]), n_pair++ & 1, a.wait_ns)",
                 "warp_wait(saddr(&s_qempty[slot]), (turn & 1) ^ 1, a.wait_ns)",
                 "warp_wait(saddr(&s_empty[s]), (x / NS & 1) ^ 1, a.wait_ns)",
                 "warp_wait(saddr(&s_tail), n_tail++ & 1, a.wait_ns)",
                 "warp_wait(saddr(&s_qfull[slot]), q_turn & 1, a.wait_ns)",
                 "ok = warp_wait(saddr(&s_full[at]), ring_turn, a.wait_ns); if (++ring_slot == NS) { ring_slot = 0; ring_turn ^= 1; }",
                 "if (!two && (j & 1) != t) { if (lane == 0) mbar_arrive(saddr(&s_empty[at])); continue; }",
                 "if (n_qk >= 2) ok = product_done(n_qk - 2);",
                 "warp_wait(saddr(&s_pready[t][n_pv & 1]), n_pv >> 1 & 1, a.wait_ns)"):
        assert CODE.count(text) == 1, text
    # Those and, at a warp's end, what it issued itself: no wait that the model does not know.
    assert len(re.findall(r"\bwarp_wait\(saddr", CODE)) == 12 + 1
    assert len(re.findall(r"\bproduct_done\(n", CODE)) == 4
