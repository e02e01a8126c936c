'use strict'
/*
 * Attention behind shared prefixes, adapters and head preparation under several
 * axes through the N-API addon and HipGpu (CommonJS, Node 12). Usage:
 *   node serving_test.js cpu    (no GPU: scratch sizes, refused arguments)
 *   node serving_test.js gpu    (against the calls that share nothing, and sums in
 *                                doubles)
 * Assertions fail the process; a JSON summary goes to stdout.
 */
const assert = require('assert')
const path = require('path')

const hip = require(path.join(__dirname, '..', '..', 'webgllm_amd', 'node', 'index.js'))

const shape = { heads: 4, kvHeads: 2, headDim: 64 }
const HD = 64
const QD = 4 * HD
const KVD = 2 * HD

function invalid (fn, text) {
  assert.throws(fn, (e) => (e instanceof hip.GpuError || e.name === 'GpuError') && e.code === 'WG_ERR_INVALID' && (!text || e.message.includes(text)))
}

function cpu () {
  const A = hip.addon
  const sizes = { pages: 9, pageSize: 16, ldTable: 4, sequences: 2 }
  const long = { pages: 9000, pageSize: 16, ldTable: 4000, sequences: 2 }
  const adapters = { slots: 3, maxRank: 16, K: 64, N: 96, cols: [64, 32] }
  for (const name of ['pagedHeadPrepAxes', 'pagedAttnShared', 'adapterAdd']) assert.throws(() => A[name]({}), TypeError)
  assert.throws(() => A.adapterScratchBytes(null, 4), TypeError)
  assert.throws(() => A.adapterScratchBytes(Object.assign({}, adapters, { cols: [1, 2, 3, 4, 5] }), 4), TypeError)
  assert.throws(() => A.adapterScratchBytes(Object.assign({}, adapters, { cols: ['x'] }), 4), TypeError)
  invalid(() => A.adapterScratchBytes(Object.assign({}, adapters, { slots: 0 }), 4), 'adapters')
  invalid(() => A.pagedSharedScratchBytes(Object.assign({}, sizes, { pages: 0 }), shape, 2, 1))
  return {
    shared: [sizes, long].map((c) => [2, 7].map((m) => A.pagedSharedScratchBytes(c, shape, m, 1))),
    adapter: [1, 50].map((m) => A.adapterScratchBytes(adapters, m)),
    one: A.adapterScratchBytes({ slots: 1, maxRank: 8, K: 4096, N: 64 }, 9)
  }
}

/** Half bits to a number. */
function half (h) {
  const e = (h >> 10) & 31
  const f = h & 1023
  const v = e === 0 ? f * 2 ** -24 : e === 31 ? (f ? NaN : Infinity) : (1 + f / 1024) * 2 ** (e - 15)
  return h & 0x8000 ? -v : v
}

function gpu () {
  const { GL } = hip
  const g = new hip.HipGpu(0)
  const bytes = (n) => g.texture(GL.R8UI, n, 1, { format: 0, type: 0, pixels: new Uint8Array(n) })
  const up = (a) => g.texture(GL.R8UI, a.byteLength, 1, { format: 0, type: 0, pixels: a })
  const raw = (t, T) => new T(g.readBytes(t, 0, t.bytes))
  let seed = 1
  const rnd = () => { // (uniform, variance 1)
    seed = (Math.imul(seed, 1103515245) + 12345) >>> 0
    return ((seed >>> 8) / (1 << 24) - 0.5) * Math.sqrt(12)
  }
  // three sequences that share the first 32 entries (pages 5 and 2)
  const lens = [37, 48, 41]
  const n = lens.length
  // (room for so many that sharing is worth it)
  const wide = 1400
  const table = [0, 7, 4].map((own) => Object.assign(new Array(wide).fill(-1), [5, 2, own]))
  const ropeRows = 1024 + 1
  const rope = new Float32Array(ropeRows * HD)
  for (let r = 0; r < ropeRows; r++) {
    for (let i = 0; i < HD / 2; i++) {
      const a = (r < 1024 ? r : (r - 1024) * 1024) * Math.pow(1e4, -2 * i / HD)
      rope[r * HD + i] = Math.cos(a)
      rope[r * HD + HD / 2 + i] = Math.sin(a)
    }
  }
  const tRope = up(rope)
  const halves = (count) => up(Uint16Array.from({ length: count }, () => 0x3000 + Math.floor(Math.abs(rnd()) * 2000) + (rnd() < 0 ? 0x8000 : 0)))
  const cache = {
    k: halves(9 * 16 * KVD), v: halves(9 * 16 * KVD), pages: 9, pageSize: 16, ldTable: wide, sequences: n,
    table: up(Int32Array.from([].concat(...table))), lens: up(Int32Array.from(lens))
  }
  // axes: rows whose positions are one number have the single-position call's bits,
  // and each frequency turns by its own axis' position
  const qkv = up(Float32Array.from({ length: n * (QD + 2 * KVD) }, rnd))
  const prep = (pos, sections, inter) => {
    const q = bytes(n * QD * 4)
    if (sections) g.ops.pagedHeadPrepAxes(qkv, n, shape, null, null, tRope, ropeRows, up(Int32Array.from([].concat(...pos))), sections, inter, cache, null, q)
    else g.ops.pagedHeadPrep(qkv, n, shape, null, null, tRope, ropeRows, up(Int32Array.from(pos)), cache, null, q)
    return raw(q, Uint32Array)
  }
  const plain = [[3, 700, 41], [9, 2, 1000]].map((p) => prep(p))
  assert.deepStrictEqual(prep([[3, 3], [700, 700], [41, 41]], [20, 12], false), plain[0])
  const mixed = prep([[3, 9], [700, 2], [41, 1000]], [16, 16], true)
  for (let i = 0; i < mixed.length; i++) assert.strictEqual(mixed[i], plain[i % (HD / 2) % 2][i])
  // the shared prefix against the decode call
  const q = up(Float32Array.from({ length: n * QD }, () => rnd() / 8))
  const groupStart = up(Int32Array.from([0, 3]))
  const shared = up(Int32Array.from([32]))
  const out = bytes(n * QD * 2)
  const out2 = bytes(n * QD * 2)
  g.ops.pagedAttnShared(q, n, shape, cache, null, groupStart, shared, 1, out, bytes(g.ops.pagedSharedScratchBytes(cache, shape, n, 1)))
  g.ops.pagedAttnDecode(q, shape, cache, 0, 0, null, out2, bytes(g.ops.pagedDecodeScratchBytes(cache, shape)))
  // Either call is off by at most 2^-11 of its output and 2^-10 of the largest
  // value (weights and sums): together under 2^-8 of it.
  const vMax = Math.max(...Array.from(raw(cache.v, Uint16Array), (h) => Math.abs(half(h))))
  const got = raw(out, Uint16Array)
  const want = raw(out2, Uint16Array)
  for (let i = 0; i < got.length; i++) assert.ok(Math.abs(half(got[i]) - half(want[i])) <= vMax / 256, `${i}`)
  const rowStart = up(Int32Array.from([0, 1, 2, 3]))
  const rowsBytes = g.ops.pagedSharedScratchBytes(cache, shape, n, 1)
  g.ops.pagedAttnShared(q, n, shape, cache, rowStart, groupStart, shared, 1, out2, rowsBytes ? bytes(rowsBytes) : null)
  const rows = raw(out2, Uint16Array)
  for (let i = 0; i < got.length; i++) assert.ok(Math.abs(half(rows[i]) - half(want[i])) <= vMax / 256, `${i}`)
  // adapters against doubles: A x by at most 66 additions of products of halves under
  // 2^-24 of their sum each, 22 bits of it kept, 16 more, 5 roundings of the result
  const K = 64
  const N = 96
  const ad = { a: halves(2 * 2 * 16 * K), b: halves(2 * N * 16), rank: up(Int32Array.from([16, 5])), scale: up(Float32Array.from([0.5, 2])), slots: 2, maxRank: 16, K, N, cols: [64, 32] }
  const x = halves(n * K)
  const y0 = Float32Array.from({ length: n * N }, rnd)
  const y = up(y0)
  const rowScale = up(Float32Array.from([1, 2, 4]))
  g.ops.adapterAdd(x, n, ad, up(Int32Array.from([1, -1, 0])), null, n, rowScale, y, bytes(g.ops.adapterScratchBytes(ad, n)))
  const [xa, aa, ba, ya] = [raw(x, Uint16Array), raw(ad.a, Uint16Array), raw(ad.b, Uint16Array), raw(y, Float32Array)]
  for (let m = 0; m < n; m++) {
    const slot = [1, -1, 0][m]
    for (let j = 0; j < N; j++) {
      let sum = 0
      let mag = 0
      for (let r = 0; slot >= 0 && r < [16, 5][slot]; r++) {
        let t = 0
        let tm = 0
        for (let k = 0; k < K; k++) {
          const p = half(aa[((slot * 2 + (j >= 64 ? 1 : 0)) * 16 + r) * K + k]) * half(xa[m * K + k])
          t += p
          tm += Math.abs(p)
        }
        const b = half(ba[(slot * N + j) * 16 + r])
        sum += t * b
        mag += tm * Math.abs(b)
      }
      const f = slot < 0 ? 0 : [0.5, 2][slot] * [1, 2, 4][m]
      const w = y0[m * N + j] + f * sum
      assert.ok(Math.abs(ya[m * N + j] - w) <= f * mag * 110 * 2 ** -24 + 2 ** -23 * Math.abs(w), `${m} ${j}`)
    }
  }
  const small = bytes(16)
  invalid(() => g.ops.pagedAttnShared(q, n, shape, cache, null, groupStart, shared, 1, out, small), 'scratch: ')
  invalid(() => g.ops.pagedAttnShared(q, n, shape, cache, null, groupStart, shared, 4, out, small), 'groupStart: ')
  invalid(() => g.ops.pagedHeadPrepAxes(qkv, n, shape, null, null, tRope, ropeRows, small, [16, 16], false, cache, null, out), 'pos: ')
  invalid(() => g.ops.pagedHeadPrepAxes(qkv, n, shape, null, null, tRope, ropeRows, qkv, [16, 15], false, cache, null, q), '31 frequencies')
  invalid(() => g.ops.adapterAdd(x, n, ad, small, null, n, null, small, bytes(4096)), 'y: ')
  invalid(() => g.ops.adapterAdd(x, n, Object.assign({}, ad, { b: small }), small, null, n, null, y, bytes(4096)), 'b: ')
  invalid(() => g.ops.adapterAdd(x, n, Object.assign({}, ad, { cols: [64, 31] }), small, null, n, null, y, bytes(4096)), '31 outputs')
  g.dispose()
  return { rows: n }
}

const out = process.argv[2] === 'cpu' ? cpu() : gpu()
process.stdout.write(JSON.stringify(out) + '\n')
