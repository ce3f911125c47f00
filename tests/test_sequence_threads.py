"""The sequence operators over packs from two host threads at once."""
import threading

import pytest
import torch

from seq_util import marks
from test_sequence import DEV, _leaf, _model, _model_inputs, _normal, spc  # noqa: F401


def _both(*work):
    """Runs the two at once and raises what either raised."""
    errors = []

    def run(f):
        try:
            f()
        except BaseException as e:  # noqa: B036
            errors.append(e)
    threads = [threading.Thread(target=run, args=(f,)) for f in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join(100)
    assert not any(t.is_alive() for t in threads)
    if errors:
        raise errors[0]


class _Library:
    """The library's size queries, and entries that launch nothing: each leaves its workspace's address (the third
    argument from the end) and waits until the other thread's has done so too."""

    def __init__(self, real):
        self.real, self.barrier, self.seen = real, threading.Barrier(2, timeout=60), []

    def __getattr__(self, name):
        if name.endswith('_bytes'):
            return getattr(self.real, name)

        def entry(*args):
            self.seen.append(args[-3])
            self.barrier.wait()
            return 0
        return entry


@pytest.mark.parametrize('which', ['layout', 'attention', 'attention backward', 'norm backward', 'recurrence',
                                   'recurrence backward'])
def test_calls_in_flight_have_scratch_of_their_own(monkeypatch, which):
    from kaolin import _native as N
    from kaolin import _sequence as S
    library = _Library(N.lib())
    monkeypatch.setattr(N, 'lib', lambda: library)
    monkeypatch.setattr(N, 'stream_of', lambda device: 0)
    monkeypatch.setattr(N, 'on_device', lambda device: N._NULL)
    monkeypatch.setattr(S, 'check_all_same_gpu', lambda func, args: None)
    n = 300
    layout = torch.zeros(n, dtype=torch.int32), torch.zeros(n + 1, dtype=torch.int32)
    q, x, lse = torch.zeros(n, 1, 8), torch.zeros(n, 8), torch.zeros(n, 1)
    call = {
        'layout': lambda: S.pack_layout_cuda(torch.zeros(n, dtype=torch.bool)),
        'attention': lambda: S.pack_attention_forward_cuda(q, q, q, layout, layout, 1.0, False, False),
        'attention backward': lambda: S.pack_attention_backward_cuda(q, q, q, q, layout, layout, q, lse, None, 1.0, False,
                                                                     True, True),
        'norm backward': lambda: S.norm_rotary_backward_cuda(q, q, q, q, None, None, torch.zeros(4, dtype=torch.float64),
                                                             layout, None, 1e-6, False, True),
        'recurrence': lambda: S.linear_recurrence_forward_cuda(x, x, layout, None, False),
        'recurrence backward': lambda: S.linear_recurrence_backward_cuda(x, x, x, layout, None, False),
    }[which]
    _both(call, call)
    assert len(library.seen) == 2 and library.seen[0] != library.seen[1]


@pytest.mark.gpu
def test_two_threads_on_one_stream(spc):
    """One thread trains, another only looks, on the same stream: every result as alone."""
    b, p, x, depth = _model_inputs(lens=(300, 1, 500, 90))
    b, x, depth = b.to(DEV), x.to(DEV), depth.to(DEV)
    names = [n for n in p if n != 'freqs']
    k = _normal(9, 4000, 1, 16).to(DEV)
    q, one = _normal(10, 1, 1, 16).to(DEV), marks([1]).to(DEV)
    whole = marks([4000]).to(DEV)
    a, y = torch.sigmoid(_normal(11, 9000, 260)).to(DEV), _normal(12, 9000, 260).to(DEV)
    long = marks([4000, 5000]).to(DEV)

    def train():
        pd = {n: _leaf(z) if n != 'freqs' else z.to(DEV) for n, z in p.items()}
        h = _model(spc, pd, x, b, depth)
        return [h.detach(), *torch.autograd.grad(h, [pd[n] for n in names], h.detach())]

    def look():
        return [spc.pack_attention(q, k, k, whole, q_boundaries=one), spc.linear_recurrence(a, y, long)]
    want, got = (train(), look()), ([], [])
    torch.cuda.synchronize()

    def many(f, results):
        for _ in range(30):
            results.append(f())
    _both(lambda: many(train, got[0]), lambda: many(look, got[1]))
    torch.cuda.synchronize()
    for w, results in zip(want, got):
        for r in results:
            for z, y0 in zip(r, w):
                assert torch.equal(z, y0)
