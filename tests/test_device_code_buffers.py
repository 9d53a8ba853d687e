"""The buffer loads to LDS that inline assembly issues keep their wait states in
the built library's gfx950 code: one after the scalar write of M0, five after a
vector instruction's SGPR result that is one of the four resource words."""
import re

from test_device_code import kernels, sgprs, wait_states


def written_sgprs(ins):
    """SGPRs that a vector instruction writes (readlanes, compares, carry-outs)."""
    ops = re.split(r"[ ,]+", ins)
    if not ops[0].startswith("v_"):
        return set()
    return sgprs(ops[1]) | (sgprs(ops[2]) if "_co_" in ops[0] and len(ops) > 2 else set())


def test_buffer_loads_to_lds_keep_their_wait_states(tmp_path):
    seen, wrong = 0, []
    for name, code in kernels(tmp_path):
        for i, ins in enumerate(code):
            if not (ins.startswith("buffer_load") and ins.endswith("lds")):
                continue
            seen += 1
            words = sgprs(re.split(r"[ ,]+", ins)[2])
            assert len(words) == 4, ins
            states = 0
            for before in reversed(code[max(0, i - 6):i]):
                ops = re.split(r"[ ,]+", before)
                if ops[0].startswith("s_") and ops[1:2] == ["m0"] and states < 1:
                    wrong.append((name, before, ins))
                if states < 5 and written_sgprs(before) & words:
                    wrong.append((name, before, ins))
                states += wait_states(before)
    assert seen, "no buffer load to LDS in the library"
    assert not wrong, wrong[:5]
