"""What tgbm_scores_sample, _feedback, _norm and _norm_backward refuse is refused before anything reaches a GPU: the pointers here are never
followed."""
import pytest

P, FAR = 1 << 20, 1 << 30   # addresses that are aligned for everything
NAN, INF = float('nan'), float('inf')


@pytest.fixture(scope='module')
def lib():
    from thundergbm_b200 import _lib
    return _lib.lib()


def _sample(lib, n=4, k=40, type=0, z=P, rs=40, cs=1, m=1, ut=0, u=P, T=1.0, Ts=None, top_k=0, ks=None, p=1.0, ps=None, q=0.0, qs=None, c=P, logs=None, every=None):
    return lib.tgbm_scores_sample(n, k, type, z, rs, cs, m, ut, u, T, Ts, top_k, ks, p, ps, q, qs, c, logs, every, None)


def _feedback(lib, n=4, k=40, type=0, z=P, rs=40, cs=1, m=1, c=P, gains=P, old=None, ref=None, w=None, T=1.0, low=1.0, high=INF, kl=0.0, b=0.0, loss=P, logs=None,
              gives=1, g=P + 65536, grs=40, gcs=1):
    return lib.tgbm_scores_feedback(n, k, type, z, rs, cs, m, c, gains, old, ref, w, T, low, high, kl, b, loss, logs, gives, g, grs, gcs, None)


def _norm(lib, n=4, k=40, type=0, z=P, rs=40, cs=1, out=P + 65536, ors=40, ocs=1, gain=None, bias=None, eps=1e-5, mean=FAR, rstd=FAR):
    return lib.tgbm_scores_norm(n, k, type, z, rs, cs, out, ors, ocs, gain, bias, eps, mean, rstd, None)


def _back(lib, n=4, k=40, type=0, g=P + 16384, grs=40, gcs=1, z=P, rs=40, cs=1, mean=FAR, rstd=FAR, gain=None, out=P + 65536, ors=40, ocs=1, tg=FAR, tb=FAR, work=FAR,
          size=1 << 30):
    return lib.tgbm_scores_norm_backward(n, k, type, g, grs, gcs, z, rs, cs, mean, rstd, gain, out, ors, ocs, tg, tb, work, size, None)


@pytest.mark.parametrize('call,args,says', [
    (_sample, dict(n=-1), 'rows'), (_sample, dict(k=0), 'classes'), (_sample, dict(k=(1 << 20) + 1), 'classes'), (_sample, dict(type=3), 'type'),
    (_sample, dict(z=None), 'null'), (_sample, dict(z=P + 2), 'aligned'), (_sample, dict(rs=-40), 'negative'), (_sample, dict(m=0), 'draws'), (_sample, dict(m=129), 'draws'),
    (_sample, dict(ut=1), 'floats or doubles'), (_sample, dict(ut=2), 'floats or doubles'), (_sample, dict(u=None), 'null'), (_sample, dict(u=P + 4, ut=3), 'aligned'),
    (_sample, dict(T=-0.5), 'temperature'), (_sample, dict(T=INF), 'temperature'), (_sample, dict(T=NAN), 'temperature'), (_sample, dict(Ts=P + 1), 'aligned'),
    (_sample, dict(top_k=-1), 'top_k'), (_sample, dict(p=1.01), 'top_p'), (_sample, dict(p=NAN), 'top_p'), (_sample, dict(q=-1e-9), 'min_p'), (_sample, dict(q=NAN), 'min_p'),
    (_sample, dict(c=None), 'null'), (_sample, dict(c=P + 2), 'aligned'), (_sample, dict(logs=P + 1), 'aligned'), (_sample, dict(every=P + 2), 'aligned'),
    (_feedback, dict(m=0), 'draws'), (_feedback, dict(T=0.0), 'temperature'), (_feedback, dict(T=4e-39), 'temperature'), (_feedback, dict(low=-0.1), 'clip'),
    (_feedback, dict(low=1.1), 'clip'), (_feedback, dict(high=-1.0), 'clip'), (_feedback, dict(high=NAN), 'clip'), (_feedback, dict(kl=-1.0, ref=P), 'kl'),
    (_feedback, dict(kl=0.1), 'reference'), (_feedback, dict(b=INF), 'entropy'), (_feedback, dict(gives=3), 'kind'), (_feedback, dict(c=None), 'null'),
    (_feedback, dict(gains=None), 'null'), (_feedback, dict(gains=P + 2), 'aligned'), (_feedback, dict(gives=0, loss=None), 'loss'), (_feedback, dict(g=None), 'null'),
    (_feedback, dict(g=P), 'share'), (_feedback, dict(gives=2, g=P + 65540), 'aligned'), (_feedback, dict(grs=1, gcs=1), 'share'), (_feedback, dict(gives=2, g=P + 8), 'share'),
    (_norm, dict(eps=0.0), 'eps'), (_norm, dict(eps=NAN), 'eps'), (_norm, dict(eps=INF), 'eps'), (_norm, dict(out=None), 'null'), (_norm, dict(out=P + 4), 'share'),
    (_norm, dict(out=P, ors=80), 'share'), (_norm, dict(ocs=0), 'share'), (_norm, dict(gain=P + 65536), 'share'), (_norm, dict(bias=P + 65536 + 636), 'share'),
    (_norm, dict(gain=FAR + 2), 'aligned'), (_norm, dict(mean=FAR + 1), 'aligned'), (_norm, dict(type=-1), 'type'),
    (_back, dict(tg=None), 'both'), (_back, dict(tb=None), 'both'), (_back, dict(work=None), 'work'), (_back, dict(size=4 * 2 * 40 - 1), 'work'),
    (_back, dict(work=FAR + 8), 'aligned'), (_back, dict(out=P), 'share'), (_back, dict(out=P + 16384), 'share'), (_back, dict(mean=None), 'null'),
    (_back, dict(rstd=None), 'null'), (_back, dict(g=None), 'null'), (_back, dict(z=None), 'null'), (_back, dict(g=P + 16385), 'aligned'),
])
def test_refused(lib, call, args, says):
    assert call(lib, **args) == 1
    assert says in lib.tgbm_last_error().decode()


@pytest.mark.parametrize('call', [_sample, _feedback, _norm])
def test_no_rows_is_nothing_to_do(lib, call):
    assert call(lib, n=0, z=None) == 0
    assert lib.tgbm_last_error() == b''


def test_work_of_the_weights_gradient(lib):
    """Enough for a partial sum per class at least, little whatever the shape."""
    for n in (1, 31, 5000, 2 ** 31 - 1):
        for k in (1, 7, 250, 8191, 65536, 1 << 20):
            assert 8 * k <= lib.tgbm_scores_norm_work(n, k) <= 160 << 20
    assert lib.tgbm_scores_norm_work(0, 5) == lib.tgbm_scores_norm_work(5, 0) == 0


@pytest.mark.parametrize('call,args', [(_sample, {}), (_feedback, dict(gives=0)), (_norm, dict(out=1 << 40, ors=131072))])
@pytest.mark.parametrize('n', [1 << 28, (1 << 31) - 1])
def test_more_blocks_than_a_launch_has_are_refused(lib, call, args, n):
    """Rows that are all the same one (stride 0) take no memory, so there may be any number of them: 8 blocks for each would be more than a launch has,
    and their number modulo 2^32 would leave rows out."""
    assert call(lib, n=n, k=131072, rs=0, **args) == 1
    assert 'rows' in lib.tgbm_last_error().decode()
