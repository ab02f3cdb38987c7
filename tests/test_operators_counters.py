"""The words that calls count their finished parts in (trellis_ops._counter_words), without a device."""
import torch


def test_threads_share_a_streams_words(monkeypatch):
    """Two threads that ask for a stream's words at the same time get one set: the other would be freed, and its
    memory given to a workspace, while a call still counts in it."""
    import trellis_ops as xt
    monkeypatch.setattr(xt, "_counters", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    zeros, won = torch.zeros, []

    def slow_zeros(*a, **kw):           # while the first thread allocates, the second comes and goes
        if not won:
            won.append(None)
            won[0] = xt._counter_words(torch.device("cpu"), 7)
        return zeros(*a, **kw)

    monkeypatch.setattr(torch, "zeros", slow_zeros)
    first = xt._counter_words(torch.device("cpu"), 7)
    assert first is won[0] and xt._counter_words(torch.device("cpu"), 7) is first
    assert xt._counter_words(torch.device("cpu"), 8) is not first
