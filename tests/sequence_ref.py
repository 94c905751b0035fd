"""Plain float64 restatements of the state-space sequence operators (pb_sed_amd.ops: causal_conv_*, selective_scan_*, layer_norm_*,
dropout) and the bounds their tests use.  Everything runs clip by clip and frame by frame on the CPU.

Bounds.  u = 2^-24 is half a step of float32.  A result is compared with |got - ref| <= eps_T / 2 |ref| + k u M, where eps_T / 2 is the one
rounding to the output's type (0 for float32 outputs: that rounding is in k), M is the MAJORANT of the result - the same formula with every
factor replaced by its absolute value, so that a sum's rounding errors are measured against what was added and not against what
is left of it - and k counts the roundings a term meets: every product and sum on its way is 1, v_exp_f32 / v_rcp_f32 are 1 ulp = 2 u, and
exp(x) computed from a product x = D A carries |x| u of that product's rounding, which exp(x) |x| <= 0.37 makes at most 1 more."""
import math

import numpy as np
import torch

U = 2. ** -24
HALF = {torch.float32: 0., torch.bfloat16: 2. ** -8, torch.float16: 2. ** -11}


def check(got, ref, major, k, what):
    """|got - ref| <= HALF |ref| + k U major + the smallest half subnormal of the type, elementwise; a value beyond the type's largest
    finite one rounds to infinity (float16: 65504)."""
    half, largest = HALF[got.dtype], torch.finfo(got.dtype).max
    got = got.detach().cpu().double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    tiny = {0.: 2. ** -126, 2. ** -8: 2. ** -126, 2. ** -11: 2. ** -25}[half]
    # (1 + half): the float32 error is rounded along with the value
    tol = half * ref.abs() + (1 + half) * k * U * major + tiny
    beyond = torch.isinf(got) & (torch.sign(got) == torch.sign(ref)) & (ref.abs() + tol >= largest)
    bad = ~(((got - ref).abs() <= tol) | beyond)
    assert not bad.any(), (what, int(bad.sum()), 'of', bad.numel(), 'worst', float(((got - ref).abs() / tol).nan_to_num(math.inf).max()),
                           'first', tuple(int(v[0]) for v in torch.nonzero(bad, as_tuple=True)))


def _order(n, reverse):
    return list(range(n))[::-1] if reverse else list(range(n))


def conv(x, w, bias, *, silu=True, seq_len=None, reverse=False, state=None, dy=None, dstate_out=None):
    """Returns a dict: y, state_out and - with dy - dx, dstate, dw, db; and the majorants under the same names in 'major'."""
    t, b, d = x.shape
    k = w.shape[1]
    out = dict(y=torch.zeros_like(x), state_out=x.new_zeros(b, k - 1, d))
    if dy is not None:
        out.update(dx=torch.zeros_like(x), dstate=x.new_zeros(b, k - 1, d), dw=torch.zeros_like(w), db=x.new_zeros(d))
    major = {key: torch.zeros_like(v) for key, v in out.items()}
    for i in range(b):
        n = t if seq_len is None else int(seq_len[i])
        order = _order(n, reverse)
        long = torch.cat([x.new_zeros(k - 1, d) if state is None else state[i], x[order, i]])
        out['state_out'][i] = long[n:]
        grad = torch.zeros_like(long)
        grad_major = torch.zeros_like(long)
        for s, f in enumerate(order):
            terms = long[s:s + k] * w.t()
            pre = terms.sum(0) + (0 if bias is None else bias)
            pre_major = terms.abs().sum(0) + (0 if bias is None else bias.abs())
            sg = torch.sigmoid(pre)
            out['y'][f, i] = pre * sg if silu else pre
            # |silu'| <= 1.1: an error of pre reaches y at most 1.1-fold; |y| <= |pre|
            major['y'][f, i] = 1.1 * pre_major
            if dy is not None:
                slope = sg * (1 + pre * (1 - sg)) if silu else torch.ones_like(pre)
                g = dy[f, i] * slope
                # the slope: |silu''| <= 0.5, and its own roundings against 1.1
                gm = dy[f, i].abs() * (1.1 + .5 * pre_major if silu else 1.)
                grad[s:s + k] += g * w.t()
                grad_major[s:s + k] += gm * w.t().abs()
                out['dw'] += (g * long[s:s + k]).t()
                major['dw'] += (gm * long[s:s + k].abs()).t()
                out['db'] += g
                major['db'] += gm
        if dy is not None:
            if dstate_out is not None:
                grad[n:] += dstate_out[i]
                grad_major[n:] += dstate_out[i].abs()
            out['dx'][order, i], major['dx'][order, i] = grad[k - 1:], grad_major[k - 1:]
            out['dstate'][i], major['dstate'][i] = grad[:k - 1], grad_major[:k - 1]
    return dict(out, major=major)


def scan(u, delta, a_log, b, c, *, d=None, z=None, delta_bias=None, softplus=True, seq_len=None, reverse=False, state=None, dy=None,
         dstate_out=None):
    """Returns a dict: y, state_out and - with dy - du, ddelta, db, dc, dz, dstate, da_log, dd, ddelta_bias; majorants in 'major'."""
    t, bs, width = u.shape
    n = a_log.shape[1]
    rate = -torch.exp(a_log)
    out = dict(y=torch.zeros_like(u), state_out=u.new_zeros(bs, width, n))
    if dy is not None:
        out.update(du=torch.zeros_like(u), ddelta=torch.zeros_like(u), db=torch.zeros_like(b), dc=torch.zeros_like(b), dz=torch.zeros_like(u),
                   dstate=u.new_zeros(bs, width, n), da_log=torch.zeros_like(a_log), dd=u.new_zeros(width), ddelta_bias=u.new_zeros(width))
    major = {key: torch.zeros_like(v) for key, v in out.items()}
    skip = u.new_zeros(width) if d is None else d
    for i in range(bs):
        length = t if seq_len is None else int(seq_len[i])
        order = _order(length, reverse)
        h = u.new_zeros(width, n) if state is None else state[i]
        hm = h.abs()
        past, steps = [], []
        for f in order:
            raw = delta[f, i] + (0 if delta_bias is None else delta_bias)
            raw_major = delta[f, i].abs() + (0 if delta_bias is None else delta_bias.abs())
            st = torch.nn.functional.softplus(raw, threshold=100) if softplus else raw
            # an error of raw moves softplus by its slope sigmoid(raw) <= softplus(raw) for the part below, 1 above
            st_major = st.abs() + (torch.sigmoid(raw) * raw_major if softplus else raw_major)
            decay = torch.exp(st[:, None] * rate)
            # decay reacts to errors of the step: |d decay| = decay |rate| d step
            decay_major = decay * (1 + st_major[:, None] * rate.abs())
            drive = st[:, None] * u[f, i][:, None] * b[f, i][None]
            drive_major = st_major[:, None] * u[f, i].abs()[:, None] * b[f, i].abs()[None]
            past.append((h, hm))
            h, hm = decay * h + drive, decay * hm + decay_major * h.abs() + drive_major
            pre = (h * c[f, i]).sum(-1) + skip * u[f, i]
            pre_major = (hm * c[f, i].abs()).sum(-1) + (skip * u[f, i]).abs()
            gate = u.new_ones(width) if z is None else z[f, i] * torch.sigmoid(z[f, i])
            out['y'][f, i], major['y'][f, i] = pre * gate, pre_major * gate.abs() + (0 if z is None else (pre * z[f, i]).abs() * .3)
            steps.append((f, raw, st, st_major, decay, decay_major, drive, drive_major, pre, pre_major, gate, h, hm))
        out['state_out'][i], major['state_out'][i] = h, hm
        if dy is None:
            continue
        r = u.new_zeros(width, n) if dstate_out is None else dstate_out[i]
        rm = r.abs()
        for (f, raw, st, stm, decay, dm, drive, drm, pre, prem, gate, h, hm), (h0, hm0) in zip(reversed(steps), reversed(past)):
            uu, bb, cc = u[f, i], b[f, i], c[f, i]
            g = dy[f, i] * gate
            gm = dy[f, i].abs() * (gate.abs() + (0 if z is None else z[f, i].abs() * .3))
            r, rm = r + g[:, None] * cc, rm + gm[:, None] * cc.abs()
            q, qm = decay * h0, decay * hm0 + dm * h0.abs()
            rb, rbm = (r * bb).sum(-1), (rm * bb.abs()).sum(-1)
            out['dc'][f, i], major['dc'][f, i] = (g[:, None] * h).sum(0), (gm[:, None] * hm).sum(0)
            out['db'][f, i], major['db'][f, i] = (r * (st * uu)[:, None]).sum(0), (rm * (stm * uu.abs())[:, None]).sum(0)
            out['du'][f, i], major['du'][f, i] = g * skip + st * rb, gm * skip.abs() + stm * rbm
            dst, dstm = uu * rb + (r * rate * q).sum(-1), uu.abs() * rbm + (rm * rate.abs() * qm).sum(-1)
            slope = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
            # sigmoid: its error against an error of raw is sigmoid(1 - sigmoid) <= sigmoid
            sm = slope * (1 + raw.abs() + delta[f, i].abs())
            out['ddelta'][f, i], major['ddelta'][f, i] = dst * slope, dstm * sm
            out['ddelta_bias'] += dst * slope
            major['ddelta_bias'] += dstm * sm
            out['da_log'] += r * rate * q * st[:, None]
            major['da_log'] += rm * rate.abs() * qm * stm[:, None]
            out['dd'] += g * uu
            major['dd'] += gm * uu.abs()
            if z is not None:
                sg = torch.sigmoid(z[f, i])
                out['dz'][f, i] = dy[f, i] * pre * sg * (1 + z[f, i] * (1 - sg))
                major['dz'][f, i] = dy[f, i].abs() * prem * (1.1 + z[f, i].abs())
            r, rm = r * decay, rm * decay + r.abs() * dm
        out['dstate'][i], major['dstate'][i] = r, rm
    return dict(out, major=major)


def layer_norm(x, w, b, eps, dy=None):
    c = x.shape[-1]
    mean = x.mean(-1, keepdim=True)
    xc = x - mean
    std = ((xc * xc).mean(-1, keepdim=True) + eps).sqrt()
    xh = xc / std
    ww, bb = (torch.ones(c, dtype=x.dtype) if w is None else w), (torch.zeros(c, dtype=x.dtype) if b is None else b)
    out = dict(y=xh * ww + bb)
    # the mean is off by the roundings of its sum (against mean |x|), which shifts a whole row of xh
    xhm = (x.abs() + x.abs().mean(-1, keepdim=True)) / std + xh.abs()
    major = dict(y=xhm * ww.abs() + bb.abs())
    if dy is not None:
        g, gm = dy * ww, (dy * ww).abs()
        out['dx'] = (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True)) / std
        cross = (gm * xhm).mean(-1, keepdim=True)
        major['dx'] = (gm + gm.mean(-1, keepdim=True) + xhm * cross + xh.abs() * cross) / std
        lead = tuple(range(x.dim() - 1))
        out['dw'], major['dw'] = (dy * xh).sum(lead), (dy.abs() * xhm).sum(lead)
        out['db'], major['db'] = dy.sum(lead), dy.abs().sum(lead)
    return dict(out, major=major)


def philox_words(seed, step, site, n, rounds=7):
    """n words of Philox-4x32 with plain Python integers."""
    m = (1 << 32) - 1
    words = []
    for block in range((n + 3) // 4):
        c = [block & m, block >> 32, step & m, site]
        k = [seed & m, (seed >> 32) & m]
        for _ in range(rounds):
            p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(q >> 32) ^ c[1] ^ k[0], q & m, (p >> 32) ^ c[3] ^ k[1], p & m]
            k = [(k[0] + 0x9E3779B9) & m, (k[1] + 0xBB67AE85) & m]
        words += c
    return np.array(words[:n], dtype=np.uint64)


def philox_words_at(seed, step, site, first, n):
    """Words first .. first + n - 1 of the same sequence."""
    m = (1 << 32) - 1
    out = []
    for i in range(first, first + n):
        c, k = [(i >> 2) & m, i >> 34, step & m, site], [seed & m, (seed >> 32) & m]
        for _ in range(7):
            p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(q >> 32) ^ c[1] ^ k[0], q & m, (p >> 32) ^ c[3] ^ k[1], p & m]
            k = [(k[0] + 0x9E3779B9) & m, (k[1] + 0xBB67AE85) & m]
        out.append(c[i & 3])
    return out
