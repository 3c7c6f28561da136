// f8Matrix over the stand-in addon: what it allocates, and what is left of it
// where the second of its two buffers cannot be allocated.
import assert from 'assert';
import {test, run} from './harness.js';
import {HipBackend, loadAddon} from '../../stratacuda_amd/src/backend.js';
import {fakeAddon} from './fake_addon.js';

const real = loadAddon();
const make = async () => {
    const addon = fakeAddon(real);
    addon.f8Bytes = (...a) => real.f8Bytes(...a);
    return {addon, b: await HipBackend.create({addon})};
};

test('an f8 matrix\'s two buffers', async () => {
    const {addon, b} = await make(), m = b.f8Matrix(130, 300, 128);
    assert.deepStrictEqual([m.codes.byteLength, m.scales.byteLength], [130 * 384, 8]);
    assert.deepStrictEqual([m.rows, m.cols, m.blockRows], [130, 300, 128]);
    assert.strictEqual(b.f8Matrix(5, 300).blockRows, 1);
    assert.strictEqual(addon.mem.size, 4);
});
test('nothing is left of a matrix whose scales cannot be allocated', async () => {
    const {addon, b} = await make(), alloc = addon.alloc, held = b.buffers.size, bytes = b.bytesAllocated;
    let calls = 0;
    addon.alloc = (...a) => { if (++calls === 2) throw Error('out of memory'); return alloc(...a); };
    assert.throws(() => b.f8Matrix(130, 300, 128), /out of memory/);
    assert.strictEqual(addon.mem.size, 0);
    assert.strictEqual(b.buffers.size, held);
    assert.strictEqual(b.bytesAllocated, bytes);
    b.f8Matrix(130, 300, 128);
    assert.strictEqual(addon.mem.size, 2);
});

run();
