"""What the C entries of the 8-bit attention refuse of a block table, before any launch; no GPU."""

from nano_infer_engine_b200 import _native


def test_c_entries_refuse_tables_without_columns_or_with_overlapping_rows():
    lib, bad = _native.lib, _native.NIE_ERR_INVALID
    fake = 4096
    head = [fake, 256, fake, 256, 2, fake, fake, fake, fake, 1, 0, 1, 4, 16, 2, 64, 4, fake]
    rows = [2, None, fake, 2]
    decode = [None, None, 2, 0.125, None, 0, 0, None, None]
    varlen = [fake, None, 2, 1, 0.125, None, 0, None, None]
    for stride, width in ((3, 0), (3, -1), (3, 4), (0, 0), (-3, 3)):
        assert lib.nie_paged_decode_kv8(*head, stride, width, *rows, *decode) == bad
        assert lib.nie_varlen_attention_kv8(*head, stride, width, *rows, *varlen) == bad
    none = [*decode[:2], 0, *decode[3:]]  # no request: nothing to do with any table that could be one
    assert lib.nie_paged_decode_kv8(*head, 5, 3, *rows, *none) == _native.NIE_OK
