"""Packed notes: notes of unequal length in one [rows, width] tensor, for `torch.ops.gzsl.packed_label_attention`,
`torch.ops.gzsl.gated_scan` and the HipOps methods of the same operators.

`note_spans([2491, 0, 800])` describes three notes lying one behind the other; `note_spans(lengths, pitch=T)` describes a padded
[B, T, width] batch seen as [B*T, width] rows (utils/helper.py's batches): the operators then leave the padding out.
"""
import torch


def note_spans(lengths, pitch=None, device='cuda'):
    """(spans [B,2] int64 on `device`, max_len, rows) for notes of the given lengths: packed back to back, or every `pitch`
    rows.  The table is a plan: build it once per batch shape, on the host, where the lengths are known."""
    n = [int(k) for k in lengths]
    if any(k < 0 for k in n):
        raise ValueError('a note length is negative')
    if pitch is not None and any(k > pitch for k in n):
        raise ValueError(f'a note is longer than the pitch {pitch}')
    rows, spans = 0, []
    for k in n:
        spans.append((rows, k))
        rows += k if pitch is None else int(pitch)
    table = torch.tensor(spans, dtype=torch.int64).reshape(-1, 2).to(device)
    return table, max(n, default=0), rows
