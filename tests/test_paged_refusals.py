"""What kd_paged_*, kd_verify_drafts and kd_distill_* refuse, on the host: no device is needed, none is touched."""
import ctypes

import pytest

import kd

FAKE = 1 << 20  # an aligned address that no check reads


def cache(**changes):
    given = dict(keys=FAKE, values=FAKE, key_scales=FAKE, value_scales=FAKE, pages=4, kv_heads=2, page_size=16, head_dim=64)
    given.update(changes)
    return kd.PagedCache(**given)


def batch(**changes):
    given = dict(table=FAKE, starts=FAKE, lengths=FAKE, sequences=1, table_columns=4, tokens=3)
    given.update(changes)
    return kd.PagedBatch(**given)


@pytest.fixture(scope="module")
def lib():
    return kd.Backend()


INVALID, UNSUPPORTED = -1, -4
ROWS = kd.strides(256, 64)

CACHES = [(dict(head_dim=32), UNSUPPORTED), (dict(head_dim=96), UNSUPPORTED), (dict(page_size=8), UNSUPPORTED),
          (dict(page_size=48), UNSUPPORTED), (dict(page_size=512), UNSUPPORTED), (dict(page_size=0), UNSUPPORTED),
          (dict(kv_heads=0), INVALID), (dict(pages=-1), INVALID), (dict(keys=None), INVALID), (dict(values=FAKE + 4), INVALID),
          (dict(key_scales=None), INVALID)]
BATCHES = [dict(sequences=-1), dict(tokens=-1), dict(table_columns=-1), dict(table=None), dict(starts=None),
           dict(lengths=None), dict(table_columns=1 << 40), dict(tokens=1 << 40)]


def calls(lib, c, b):
    yield lib.lib.kd_paged_append(kd.F32, c, b, None, FAKE + 64, FAKE, ROWS, 4, FAKE, ROWS, FAKE, ROWS)
    yield lib.lib.kd_paged_read(kd.F32, FAKE, FAKE, c, b)
    yield lib.lib.kd_paged_attention(kd.F32, FAKE + 64, FAKE, ROWS, 4, c, b, 1.0, 64, None, 0)


@pytest.mark.parametrize("changes,status", CACHES, ids=[str(c[0]) for c in CACHES])
def test_bad_caches(lib, changes, status):
    for rc in calls(lib, cache(**changes), batch()):
        assert rc == status and lib.error().startswith("kd_paged_")


@pytest.mark.parametrize("changes", BATCHES, ids=[str(b) for b in BATCHES])
def test_bad_batches(lib, changes):
    for rc in calls(lib, cache(), batch(**changes)):
        assert rc == INVALID and lib.error().startswith("kd_paged_")


def test_nothing_to_do_is_no_error(lib):
    for changes in (dict(sequences=0), dict(tokens=0)):
        for rc in calls(lib, cache(), batch(**changes)):
            assert rc == 0
    assert lib.lib.kd_verify_drafts(kd.F32, None, None, None, None, None, None, None, 0, 3, 10) == 0
    assert lib.lib.kd_distill_rows(kd.F32, None, None, None, None, None, 0, 5, 2, 1.0) == 0
    assert lib.lib.kd_distill_grad(kd.F64, None, None, None, None, None, None, 0, 5, 2, 1.0) == 0


def test_bad_appends(lib):
    f = lib.lib.kd_paged_append
    c, b = cache(), batch()
    good = [kd.F32, c, b, None, FAKE + 64, FAKE, ROWS, 4, FAKE, ROWS, FAKE, ROWS]
    for at, value, status in ((0, kd.F64, UNSUPPORTED), (1, None, INVALID), (2, None, INVALID), (4, None, INVALID),
                              (5, None, INVALID), (4, FAKE + 4, INVALID), (6, None, INVALID), (7, 3, INVALID), (7, 0, INVALID),
                              (8, None, INVALID), (9, None, INVALID), (9, kd.strides(-1, 64), INVALID),
                              (11, kd.strides(1 << 50, 64), INVALID), (10, FAKE + 2, INVALID)):
        args = list(good)
        args[at] = value
        if at == 4 and value == FAKE + 4:
            args[5] = FAKE
        assert f(*args) == status, (at, value)
    same = list(good)
    same[4] = same[5] = FAKE
    assert f(*same) == INVALID  # q_out is q
    for turn in (kd.Rotation(FAKE, FAKE, 9, 3, 0), kd.Rotation(FAKE, FAKE, 9, 66, 0), kd.Rotation(FAKE, FAKE, 9, -2, 0),
                 kd.Rotation(None, FAKE, 9, 4, 0), kd.Rotation(FAKE, FAKE, -1, 4, 0), kd.Rotation(FAKE, FAKE, 9, 4, 2)):
        args = list(good)
        args[3], args[4] = turn, FAKE + 64
        assert f(*args) == INVALID


def test_bad_attention(lib):
    f = lib.lib.kd_paged_attention
    good = [kd.F32, FAKE + 64, FAKE, ROWS, 4, cache(), batch(), 1.0, 64, None, 0]
    for at, value, status in ((0, kd.I64, UNSUPPORTED), (1, None, INVALID), (1, FAKE + 8, INVALID), (2, None, INVALID),
                              (3, None, INVALID), (4, 5, INVALID), (7, float("nan"), INVALID), (7, float("inf"), INVALID),
                              (8, -1, INVALID), (10, 64, INVALID), (10, -1, INVALID), (9, FAKE + 4, INVALID)):
        args = list(good)
        args[at] = value
        assert f(*args) == status, (at, value)
    n = ctypes.c_int64()
    g = lib.lib.kd_paged_attention_workspace
    assert g(None, 4, 2, 64, 1, 3, 64) == INVALID and g(ctypes.byref(n), 5, 2, 64, 1, 3, 64) == INVALID
    assert g(ctypes.byref(n), 4, 2, 64, 1, 3, 64) == 0 and n.value >= 0


def test_bad_verifications(lib):
    f = lib.lib.kd_verify_drafts
    good = [kd.F32, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 2, 3, 10]
    for at, value, status in ((0, kd.I64, UNSUPPORTED), (1, None, INVALID), (2, None, INVALID), (3, None, INVALID),
                              (5, None, INVALID), (6, None, INVALID), (7, None, INVALID), (8, -1, INVALID), (9, -1, INVALID),
                              (10, 0, INVALID), (10, 1 << 31, INVALID)):
        args = list(good)
        args[at] = value
        assert f(*args) == status, (at, value)


def test_bad_distillations(lib):
    rows, grad = lib.lib.kd_distill_rows, lib.lib.kd_distill_grad
    for good, f, sizes in (([kd.F32] + [FAKE] * 5 + [2, 9, 3, 1.0], rows, 6), ([kd.F32] + [FAKE] * 6 + [2, 9, 3, 1.0], grad, 7)):
        wrong = [(0, kd.BOOL, UNSUPPORTED), (sizes, -1, INVALID), (sizes + 1, 0, INVALID), (sizes + 2, 0, INVALID),
                 (sizes + 2, 1025, INVALID), (sizes + 3, 0.0, INVALID), (sizes + 3, float("nan"), INVALID), (sizes + 3, 1e-7, INVALID), (sizes + 3, 1e7, INVALID),
                 (sizes + 3, float("inf"), INVALID)] + [(at, None, INVALID) for at in range(1, sizes)]
        for at, value, status in wrong:
            args = list(good)
            args[at] = value
            assert f(*args) == status, (at, value)


def test_more_workgroups_than_a_launch_takes(lib):
    """Refused before a launch whose work items would not fit 32 bits."""
    assert lib.lib.kd_verify_drafts(kd.F32, *[FAKE] * 7, 1 << 22, 3, 10) == INVALID
    for cols, rows in ((96, 1 << 26), (1024, 1 << 26), (1025, 1 << 24)):
        assert lib.lib.kd_distill_rows(kd.F32, *[FAKE] * 5, rows, cols, 3, 1.0) == INVALID
        assert lib.lib.kd_distill_grad(kd.F32, *[FAKE] * 6, rows, cols, 3, 1.0) == INVALID
    c, b = cache(kv_heads=4096), batch(sequences=1 << 23)
    assert lib.lib.kd_paged_append(kd.F32, c, b, None, FAKE + 64, FAKE, ROWS, 4096, FAKE, ROWS, FAKE, ROWS) == INVALID
    assert lib.lib.kd_paged_read(kd.F32, FAKE, FAKE, c, b) == INVALID
    assert lib.lib.kd_paged_attention(kd.F32, FAKE + 64, FAKE, ROWS, 4096, c, b, 1.0, 64, None, 0) == INVALID


def test_workspaces_of_the_largest_calls(lib):
    """As many rows as a call takes have a size that is one, more have none; the part sizes follow the split's own rule."""
    n, g = ctypes.c_int64(), lib.lib.kd_paged_attention_workspace
    assert g(ctypes.byref(n), 4096, 4096, 128, 1, 1 << 19, 64) == INVALID
    assert g(ctypes.byref(n), 4096, 1, 128, 1, (1 << 19) - 1, 1 << 62) == 0 and n.value > 0
    rows = ((1 << 19) - 1) * 4096
    assert n.value % (rows * (128 + 2) * 4) == 0
    for sequences, tokens in ((0, 0), (5, 0), (1 << 23, 1)):
        assert g(ctypes.byref(n), 8, 2, 64, sequences, tokens, 1 << 20) == 0 and n.value >= 0
