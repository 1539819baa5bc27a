"""Oracle of gs_localization_amd.map_optimizer in 64 bits (numpy): TEST INFRASTRUCTURE, nothing in the product imports it.

Written from the definitions: the clipped norm, AdamW (decoupled weight decay), the 8-bit moments (a root on a grid of sixteenths of
its binade inside a window of sixteen binades per 256 elements, a ratio in 127 steps of its largest possible value, both rounded
by given random bits) and the eviction of the rows with the least accumulated weight."""
import math

import numpy as np

WINDOW = 256
M32 = 0xFFFFFFFF


def norm(grads, max_norm):
    n = math.sqrt(sum(float(np.sum(np.asarray(g, np.float64) ** 2)) for g in grads))
    return n, min(1.0, max_norm / (n + 1e-6)) if n == n else n


def span(b1, b2):
    """The largest |m| / sqrt(v): m = (1-b1) sum b1^k g_k, v = (1-b2) sum b2^k g_k^2, Cauchy-Schwarz with weights (b1 / sqrt(b2))^k."""
    return (1 - b1) / math.sqrt((1 - b2) * (1 - b1 * b1 / b2))


def adamw(p, g, m, v, t, lr, betas, eps, decay, coef=1.0):
    """One step in 64 bits; t counts from 1.  Returns p, m, v and the scale of the update's terms (for error bounds)."""
    p, g, m, v = (np.asarray(x, np.float64) for x in (p, g, m, v))
    b1, b2 = betas
    g = g * coef
    size = np.abs(m) * b1 + np.abs(g) * (1 - b1)
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    den = np.sqrt(v / (1 - b2 ** t)) + eps
    rate = lr / (1 - b1 ** t)
    with np.errstate(divide="ignore", invalid="ignore"):
        return p * (1 - lr * decay) - rate * m / den, m, v, rate * size / den


def mix(x):
    x = np.asarray(x, np.uint64)
    x = ((x ^ (x >> np.uint64(16))) * np.uint64(0x6C8E9CF5)) & np.uint64(M32)
    x = ((x ^ (x >> np.uint64(15))) * np.uint64(0x2F7A5D1B)) & np.uint64(M32)
    return x ^ (x >> np.uint64(16))


def dither(index, seed, place, t):
    """Random bits of the elements `index` of the tensor at `place` of the list in step t: 19 and 13 of them."""
    index = np.asarray(index, np.uint64)
    key = mix((t + seed * 0x9E3779B1 + (place + 1) * 0x85EBCA77) & M32)
    j = index >> np.uint64(2)
    h = mix((((((j & np.uint64(M32)) * np.uint64(0x9E3779B1)) & np.uint64(M32)) ^ key) + (j >> np.uint64(32)) * np.uint64(0x85EBCA77)) & np.uint64(M32))
    odd = np.array([1, 0xB5297A4D, 0x68E31DA5, 0x1B56C4E9], np.uint64)[(index & np.uint64(3)).astype(int)]
    r = (h * odd) & np.uint64(M32)
    r ^= r >> np.uint64(15)
    return (r >> np.uint64(13)).astype(np.int64), (r & np.uint64(8191)).astype(np.int64)


def grid_value(place):
    """The place-th value of the grid of floats with four bits of mantissa (place 0 is 0; the first binade is denormal)."""
    place = np.asarray(place, np.float64)
    binade = np.floor(place / 16)
    return np.where(binade > 0, (1 + place / 16 - binade) * 2.0 ** (binade - 127), place / 16 * 2.0 ** -126)


def grid_place(u):
    """The (fractional) place of u >= 0 on that grid."""
    u = np.asarray(u, np.float64)
    e = np.floor(np.log2(np.maximum(u, 2.0 ** -126)))
    e = np.where(2.0 ** (e + 1) <= u, e + 1, np.where(2.0 ** e > np.maximum(u, 2.0 ** -126), e - 1, e))
    return np.where(u < 2.0 ** -126, u / 2.0 ** -126 * 16, (u / 2.0 ** e - 1 + (e + 127)) * 16)


def per_block(x, n):
    return np.repeat(np.asarray(x, np.int64), WINDOW)[:n]


def decode(codes, window):
    codes = np.asarray(codes, np.int64).reshape(-1)
    return np.where(codes > 0, grid_value(codes + 16 * per_block(window, codes.size) + 1), 0.0)


def window_of(place):
    """Windows of the blocks whose largest roots have these (whole) places: the largest one's binade is the last but one."""
    place = np.asarray(place, np.int64)
    pad = np.zeros(-place.size % WINDOW, np.int64)
    return np.maximum(np.concatenate((place, pad)).reshape(-1, WINDOW).max(1) // 16 - 15, 0)


def recode(u, window):
    """Codes of roots that lie on the grid in given windows; what lies under a window becomes its lowest value."""
    place = np.rint(grid_place(u)).astype(np.int64)
    return np.where(place > 0, np.clip(place - 16 * per_block(window, place.size) - 1, 1, 255), 0)


def adamw8(p, g, rms, ratio, window, t, lr, betas, eps, decay, coef, seed, place, state_betas=None):
    """One step on 8-bit moments in 64 bits: p, then the FRACTIONAL places of the new roots and ratios with their random bits added (whose
    floors are what is stored), and the scales for error bounds.  state_betas: those that the ratios were stored with, if others."""
    u = decode(rms, window)
    m = np.asarray(ratio, np.float64).reshape(-1) / 127 * span(*(state_betas or betas)) * u
    p1, m1, v1, scale = adamw(np.asarray(p).reshape(-1), np.asarray(g).reshape(-1), m, u * u, t, lr, betas, eps, decay, coef)
    du, dr = dither(np.arange(u.size), seed, place, t)
    return p1, m1, np.sqrt(v1), grid_place(np.sqrt(v1)) + du / 2.0 ** 19, dr / 8192.0, scale


def evict(scores, keep, recent=0, weights=None, decay=1.0):
    with np.errstate(invalid="ignore"):          # (inf * 0)
        s = np.asarray(scores, np.float64) * decay
    if weights is not None and len(weights):
        s = s + np.asarray(weights, np.float64).sum(0)
    s = s.astype(np.float32)
    old = s.size - recent
    key = np.where(np.isnan(s[:old]), -np.inf, s[:old]).astype(np.float64)
    order = np.lexsort((np.arange(old), -key))          # by falling score, then by rising index
    kept = np.concatenate((np.sort(order[: keep - recent]), np.arange(old, s.size)))
    return kept.astype(np.int64), s[kept]
